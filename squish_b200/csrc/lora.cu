// lora.cu — low-rank adapters of many requests at once beside a shared projection.
//
//   out[t] = y[t] + scale[s] * B_s (A_s x[t])       s = adapter slot of row t (none: out[t] = y[t])
// optionally followed by the SiLU(gate) * up epilogue over [gate 64 | up 64] column blocks.
//
// The plan (lora_plan, once per step, shared by every projection) sorts the rows by slot, stable, and
// cuts them into tiles of at most tm rows of one adapter: 16 rows for steps of up to 512 rows, where an
// adapter has few, 128 for larger ones.
//
// The work is bound by bytes (y and out dominate): per row and projection 2 r (K + N) flops against
// 2 (K + 2 N) bytes. Up to 512 rows a cluster computes a tile in one launch (lora_row16_kernel, 6 us for
// one row of a 3584 x 3584 projection); larger steps take two (lora_shrink128_kernel,
// lora_expand128_kernel).
//
// h = scale A_s x is held in fp32 and enters the second product as a sum of two bf16 (upper and lower
// part, 16 bits of h): out is rounded once, as the formula would be; one bf16 alone would add an error
// of 2^-9 |h| per rank to every column. The rank is small, so the second product costs no time.
#include <cooperative_groups.h>

#include <type_traits>

#include "kernels.h"
#include "launch.cuh"
#include "sm100.cuh"
#include "step_ops.h"

namespace cg = cooperative_groups;

namespace sq {

namespace {

// ---------------------------------------------------------------- plan
constexpr int kPlanThreads = 1024;
constexpr int kPlanWarps = kPlanThreads / 32;

// One CTA. Warp w owns the w-th contiguous part of the rows and counts it per slot; prefix sums over
// the slots, then over the warps of a slot, give every warp its first position per slot, and a second
// walk in row order hands the positions out: a stable counting sort with no atomics between warps.
__global__ void __launch_bounds__(kPlanThreads) lora_plan_kernel(const LoraPlanParams p) {
  pdl_wait();
  pdl_trigger();
  extern __shared__ int sh[];
  const int S = p.slots + 1;       // the last group: rows without an adapter
  int* cnt = sh;                   // [warps][S]
  int* start = sh + kPlanWarps * S;  // [S + 1]
  int* tstart = start + S + 1;     // [S + 1]
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  for (int i = tid; i < kPlanWarps * S; i += kPlanThreads) cnt[i] = 0;
  __syncthreads();
  const int per = (p.M + kPlanWarps - 1) / kPlanWarps;
  const int r0 = min(p.M, warp * per), r1 = min(p.M, r0 + per);
  int* mine = cnt + warp * S;
  bool bad = false;
  auto group = [&](int r) -> int {
    const int s = p.row_slot[r];
    if (s >= p.slots || s < -1) bad = true;
    return s < 0 || s >= p.slots ? p.slots : s;
  };
  for (int r = r0 + lane; r < r1; r += 32) atomicAdd(mine + group(r), 1);
  __syncthreads();
  for (int s = tid; s < S; s += kPlanThreads) {  // per slot: exclusive prefix over the warps
    int o = 0;
    for (int w = 0; w < kPlanWarps; ++w) {
      const int c = cnt[w * S + s];
      cnt[w * S + s] = o;
      o += c;
    }
    start[s + 1] = o;
    tstart[s + 1] = (o + p.tm - 1) / p.tm;
  }
  if (tid == 0) start[0] = tstart[0] = 0;
  __syncthreads();
  if (warp == 0) {  // inclusive prefix over the slots
    int c0 = 0, c1 = 0;
    for (int s = 0; s < S; s += 32) {
      int a = s + lane < S ? start[s + lane + 1] : 0, b = s + lane < S ? tstart[s + lane + 1] : 0;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int u = __shfl_up_sync(0xffffffffu, a, o), v = __shfl_up_sync(0xffffffffu, b, o);
        if (lane >= o) {
          a += u;
          b += v;
        }
      }
      if (s + lane < S) {
        start[s + lane + 1] = a + c0;
        tstart[s + lane + 1] = b + c1;
      }
      c0 += __shfl_sync(0xffffffffu, a, 31);
      c1 += __shfl_sync(0xffffffffu, b, 31);
    }
  }
  __syncthreads();
  for (int r = r0; r < r1; r += 32) {
    const bool on = r + lane < r1;
    const int s = on ? group(r + lane) : -1;
    const unsigned same = __match_any_sync(0xffffffffu, s);
    const int before = __popc(same & ((1u << lane) - 1u));
    int base = 0;
    if (on) base = mine[s];
    __syncwarp();
    if (on) {
      p.order[start[s] + base + before] = r + lane;
      if (before == 0) mine[s] = base + __popc(same);
    }
    __syncwarp();
  }
  const int nt = min(tstart[S], p.max_tiles);
  for (int i = tid; i < nt; i += kPlanThreads) {
    int lo = 0, hi = S - 1;  // the slot of tile i: the first whose inclusive tile count exceeds i
    while (lo < hi) {
      const int mid = (lo + hi) >> 1;
      if (tstart[mid + 1] <= i) lo = mid + 1;
      else hi = mid;
    }
    const int a = start[lo] + (i - tstart[lo]) * p.tm;
    p.tiles[i] = make_int4(lo == p.slots ? -1 : lo, a, min(p.tm, start[lo + 1] - a), 0);
  }
  if (tid == 0) *p.num_tiles = nt;
  if (bad) atomicCAS(p.status, 0, SQ_ERR_BOUNDS);
}

// ---------------------------------------------------------------- y + scale B (A x)
constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;

__device__ __forceinline__ void mma16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                         uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}
__device__ __forceinline__ float lo_f(uint32_t w) { return __uint_as_float(w << 16); }
__device__ __forceinline__ float hi_f(uint32_t w) { return __uint_as_float(w & 0xffff0000u); }
// silu(g) * u with the hardware's exponential and reciprocal (2 and 1 ulp). Below g = -87 the
// reciprocal is flushed to 0; the product it replaces is smaller than 1.1e-36 |u|.
__device__ __forceinline__ float silu_mul(float g, float u) {
  float e, r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(-1.4426950408889634f * g));
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.f + e));
  return g * r * u;
}
__device__ __forceinline__ void prefetch_l2(const void* p) { asm volatile("prefetch.global.L2 [%0];" ::"l"(p)); }
// y added to the accumulators of 16 rows x 32 columns: a lane's 8 columns of its two rows.
__device__ __forceinline__ void add_to(float (&acc)[4][4], uint4 y0, uint4 y1) {
  const uint32_t w0[4] = {y0.x, y0.y, y0.z, y0.w}, w1[4] = {y1.x, y1.y, y1.z, y1.w};
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    acc[j][0] += lo_f(w0[j]);
    acc[j][1] += hi_f(w0[j]);
    acc[j][2] += lo_f(w1[j]);
    acc[j][3] += hi_f(w1[j]);
  }
}
// A lane's 8 output columns of row r (0, 1), rounded once.
template <bool SILU, int G>
__device__ __forceinline__ uint4 finish(const float (&acc)[G][4][4], int r) {
  uint32_t o[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const float a = acc[0][j][2 * r], b = acc[0][j][2 * r + 1];
    o[j] = SILU ? pack_bf16(silu_mul(a, acc[G - 1][j][2 * r]), silu_mul(b, acc[G - 1][j][2 * r + 1])) : pack_bf16(a, b);
  }
  return make_uint4(o[0], o[1], o[2], o[3]);
}

// One rank step of the expand for 16 rows x 32 columns: the lower part of h, then the upper. The four
// tiles' products alternate, so that no product waits for the one before it.
template <int R>
__device__ __forceinline__ void expand_step(float (&acc)[4][4], const uint4 (&lo)[2], const uint4 (&hi)[2],
                                            const uint4 (&w)[4]) {
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const uint4 a0 = h ? hi[0] : lo[0], a1 = h ? hi[1] : lo[1];
#pragma unroll
    for (int j = 0; j < 4; ++j) mma16816(acc[j], a0.x, a1.x, a0.y, a1.y, w[j].x, w[j].y);
    if (R != 16) {
#pragma unroll
      for (int j = 0; j < 4; ++j) mma16816(acc[j], a0.z, a1.z, a0.w, a1.w, w[j].z, w[j].w);
    }
  }
}

// Tiles of 16 rows (decode). R: padded rank of the pool. A cluster of C CTAs per tile: each takes 1/C of
// K and computes its share of h (16 x R) with mma.sync, the shares meet through the cluster's shared
// memory, and each CTA then takes 1/C of the columns; h never leaves the cluster. A decode tile holds
// one to a few rows, so what counts is latency and the bytes of A and B (64 rows over 32 adapters, K
// 3584, N 4608, rank 16: 7.9 MB, 7.2 us, of which the chain of launch, plan, x and A, exchange, B and y is
// some 6). Operands go straight from global memory into fragments: the order of k within a 32-value
// step is free as long as both operands agree, so a lane takes 8 consecutive values (16 bytes) of its
// row, and the columns of four 8-wide tiles are interleaved so that a lane's accumulators are 8
// consecutive columns of out (16-byte loads of y, 16-byte stores of out).
template <int R, bool SILU>
__global__ void __launch_bounds__(kThreads) lora_row16_kernel(const LoraParams p) {
  constexpr int RT = R / 8;           // 8-wide rank tiles
  constexpr int KW = kWarps;          // the warps split K (shrink), then the columns (expand)
  constexpr int ROWS = 16;
  constexpr int PS = R + 4;           // row stride of the fp32 shares (4: rows on distinct banks)
  constexpr int HS = R + 8;           // row stride of the bf16 parts of h
  pdl_wait();
  pdl_trigger();
  // (loads that need not wait for one another are issued together: a decode tile is a chain of waits)
  const int nt = *p.num_tiles;
  const int4 tile = p.tiles[blockIdx.x];
  if ((int)blockIdx.x >= nt) return;  // the whole cluster
  const int slot = tile.x, cnt = tile.z;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int g = lane >> 2, t = lane & 3;
  const int row0 = g < cnt ? p.order[tile.y + g] : -1, row1 = g + 8 < cnt ? p.order[tile.y + g + 8] : -1;
  const int fetch = (tid >> 4) < cnt ? p.order[tile.y + (tid >> 4)] : -1;
  const int rank = slot >= 0 ? p.rank[slot] : 0;
  const float sc = slot >= 0 ? p.scale[slot] : 0.f;
  if (rank <= 0 && p.in_place) return;
  extern __shared__ __align__(16) uint8_t smem[];
  float* part = reinterpret_cast<float*>(smem);                                    // [KW][ROWS][PS]
  __nv_bfloat16* hh = reinterpret_cast<__nv_bfloat16*>(part + KW * ROWS * PS);     // [2][ROWS][HS]
  cg::cluster_group cl = cg::this_cluster();
  const int C = gridDim.z, cr = blockIdx.z;
  const int kw = warp;
  const int live = R == 16 ? 16 : min(R, (rank + 15) / 16 * 16);  // ranks computed: whole 16-wide steps

  // this CTA's columns, in units of 32 output columns; its part of B (consecutive rows) and of y goes on
  // its way to L2 while h is computed
  constexpr int G = SILU ? 2 : 1;  // column groups of a unit (gate and up)
  const int units = SILU ? p.N / 64 : (p.N + 31) / 32;
  const int cols = C * gridDim.y, cc = blockIdx.y * C + cr;  // CTAs over the columns, this one
  const int u0 = (int)((long long)units * cc / cols), u1 = (int)((long long)units * (cc + 1) / cols);
  const __nv_bfloat16* bs = p.b + (size_t)(slot < 0 ? 0 : slot) * p.N * R;
  {
    const int n0 = u0 * 32 * G, n1 = min(p.N, u1 * 32 * G);
    if (rank > 0)
      for (size_t e = (size_t)n0 * R + tid * 64; e < (size_t)n1 * R; e += kThreads * 64) prefetch_l2(bs + e);
    if (fetch >= 0)
      for (int c = n0 + (tid & 15) * 64; c < n1; c += 16 * 64) prefetch_l2(p.y + fetch * p.ldy + c);
  }

  if (rank > 0) {
    // ---- h share: this warp's 32-wide steps of K
    float acc[RT][4];
#pragma unroll
    for (int i = 0; i < RT; ++i) acc[i][0] = acc[i][1] = acc[i][2] = acc[i][3] = 0.f;
    const int steps = (p.K + 31) / 32, parts = C * KW, me = cr * KW + kw;
    const int c0 = (int)((long long)steps * me / parts), c1 = (int)((long long)steps * (me + 1) / parts);
    const __nv_bfloat16* x0 = p.x + (row0 >= 0 ? row0 : 0) * p.ldx + t * 8;
    const __nv_bfloat16* x1 = p.x + (row1 >= 0 ? row1 : 0) * p.ldx + t * 8;
    const __nv_bfloat16* as = p.a + (size_t)slot * R * p.K + (size_t)g * p.K + t * 8;
    const uint4 zero = make_uint4(0, 0, 0, 0);
    constexpr int U = 4;
    for (int c = c0; c < c1; c += U) {
      uint4 v0[U], v1[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int k = (c + u) * 32;
        const bool in = c + u < c1 && k + t * 8 < p.K;
        v0[u] = in && row0 >= 0 ? *reinterpret_cast<const uint4*>(x0 + k) : zero;
        v1[u] = in && row1 >= 0 ? *reinterpret_cast<const uint4*>(x1 + k) : zero;
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int k = (c + u) * 32;
        const bool in = c + u < c1 && k + t * 8 < p.K;
#pragma unroll
        for (int i = 0; i < RT; ++i) {
          if (i * 8 >= live) break;
          const uint4 w = in ? __ldg(reinterpret_cast<const uint4*>(as + (size_t)i * 8 * p.K + k)) : zero;
          mma16816(acc[i], v0[u].x, v1[u].x, v0[u].y, v1[u].y, w.x, w.y);
          mma16816(acc[i], v0[u].z, v1[u].z, v0[u].w, v1[u].w, w.z, w.w);
        }
      }
    }
    float* pw = part + (size_t)kw * ROWS * PS;
#pragma unroll
    for (int i = 0; i < RT; ++i) {
      if (i * 8 >= live) break;
      *reinterpret_cast<float2*>(pw + g * PS + i * 8 + 2 * t) = make_float2(acc[i][0], acc[i][1]);
      *reinterpret_cast<float2*>(pw + (g + 8) * PS + i * 8 + 2 * t) = make_float2(acc[i][2], acc[i][3]);
    }
    __syncthreads();
    // ---- the CTA's share: sum over its K warps, in order, into part[0]
    const int nv = live / 4;
    for (int i = tid; i < ROWS * nv; i += kThreads) {
      float* q = part + (size_t)(i / nv) * PS + (i % nv) * 4;
      float4 s = *reinterpret_cast<float4*>(q);
#pragma unroll
      for (int w = 1; w < KW; ++w) {
        const float4 v = *reinterpret_cast<const float4*>(q + (size_t)w * ROWS * PS);
        s.x += v.x;
        s.y += v.y;
        s.z += v.z;
        s.w += v.w;
      }
      *reinterpret_cast<float4*>(q) = s;
    }
    cl.sync();
    // ---- h of the tile: sum of the CTAs' shares, in rank order; scaled, split into two bf16
    for (int i = tid; i < ROWS * nv; i += kThreads) {
      const int r = i / nv, c = (i % nv) * 4;
      float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
      for (int q = 0; q < C; ++q) {
        const float4 v = *reinterpret_cast<const float4*>(cl.map_shared_rank(part, q) + (size_t)r * PS + c);
        s.x += v.x;
        s.y += v.y;
        s.z += v.z;
        s.w += v.w;
      }
      s.x *= sc;
      s.y *= sc;
      s.z *= sc;
      s.w *= sc;
      const uint32_t h01 = pack_bf16(s.x, s.y), h23 = pack_bf16(s.z, s.w);
      *reinterpret_cast<uint2*>(hh + r * HS + c) = make_uint2(h01, h23);
      *reinterpret_cast<uint2*>(hh + (ROWS + r) * HS + c) =
          make_uint2(pack_bf16(s.x - lo_f(h01), s.y - hi_f(h01)), pack_bf16(s.z - lo_f(h23), s.w - hi_f(h23)));
    }
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");  // (waited for at the end)
    __syncthreads();
  }

  // ---- out = y + h B^T over this CTA's columns
  constexpr int KS = R == 16 ? 1 : R / 32;  // rank steps (32 wide; one of 16 for R = 16)
  uint4 fa[2][KS][2];                       // [upper / lower][step][row g / g + 8]
  if (rank > 0) {
#pragma unroll
    for (int q = 0; q < 2; ++q)
#pragma unroll
      for (int ks = 0; ks < KS; ++ks)
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          const __nv_bfloat16* src = hh + (size_t)(q * ROWS + g + 8 * r) * HS;
          if (R == 16) {
            const uint2 v = *reinterpret_cast<const uint2*>(src + t * 4);
            fa[q][ks][r] = make_uint4(v.x, v.y, 0, 0);
          } else if (ks * 32 + t * 8 < live) {
            fa[q][ks][r] = *reinterpret_cast<const uint4*>(src + ks * 32 + t * 8);
          } else {
            fa[q][ks][r] = make_uint4(0, 0, 0, 0);
          }
        }
  }
  for (int u = u0 + kw; u < u1; u += KW) {
    float acc[G][4][4];
    uint4 yv[G][2];  // loaded first, added last: the products do not wait for it
#pragma unroll
    for (int q = 0; q < G; ++q) {
      // first of the 32 columns of y / B: plain, or the gate / up half of block u / 2
      const int col = SILU ? (u >> 1) * 128 + q * 64 + (u & 1) * 32 : u * 32;
      const bool in = SILU || col + t * 8 < p.N;
      yv[q][0] = in && row0 >= 0 ? *reinterpret_cast<const uint4*>(p.y + row0 * p.ldy + col + t * 8) : make_uint4(0, 0, 0, 0);
      yv[q][1] = in && row1 >= 0 ? *reinterpret_cast<const uint4*>(p.y + row1 * p.ldy + col + t * 8) : make_uint4(0, 0, 0, 0);
#pragma unroll
      for (int j = 0; j < 4; ++j) acc[q][j][0] = acc[q][j][1] = acc[q][j][2] = acc[q][j][3] = 0.f;
      if (rank > 0) {
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
          if (R != 16 && ks * 32 >= live) break;
          uint4 w[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const int n = col + (g >> 1) * 8 + 2 * j + (g & 1);  // (g, j) -> column: a lane's 4 tiles are 8 columns
            w[j] = make_uint4(0, 0, 0, 0);
            if (SILU || n < p.N) {
              if (R == 16) {
                const uint2 v = __ldg(reinterpret_cast<const uint2*>(bs + (size_t)n * R + t * 4));
                w[j].x = v.x;
                w[j].y = v.y;
              } else {
                w[j] = __ldg(reinterpret_cast<const uint4*>(bs + (size_t)n * R + ks * 32 + t * 8));
              }
            }
          }
          expand_step<R>(acc[q], fa[1][ks], fa[0][ks], w);
        }
      }
    }
#pragma unroll
    for (int q = 0; q < G; ++q) add_to(acc[q], yv[q][0], yv[q][1]);
    const int oc = u * 32 + t * 8;
    if (SILU || oc < p.N) {
      if (row0 >= 0) *reinterpret_cast<uint4*>(p.out + row0 * p.ldo + oc) = finish<SILU, G>(acc, 0);
      if (row1 >= 0) *reinterpret_cast<uint4*>(p.out + row1 * p.ldo + oc) = finish<SILU, G>(acc, 1);
    }
  }
  // peers may have read this CTA's share until now
  if (rank > 0) asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// ---------------------------------------------------------------- tiles of 128 rows (prefill)
__device__ __forceinline__ void cp16(void* dst, const void* src, bool on) {  // 16 bytes, or zeros
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(dst)), "l"(src), "r"(on ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
// Offset of 16-byte chunk c (0..7) of row r in a tile of 128-byte rows, 128-byte swizzle (the tensor
// cores' operand layout; a row-per-lane read meets no bank twice either).
__device__ __forceinline__ int sw(int r, int c) { return r * 128 + ((c ^ (r & 7)) << 4); }
__device__ __forceinline__ uint8_t* align1k(uint8_t* p) {
  return reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(p) + 1023) & ~uintptr_t(1023));
}

// Two launches. The shrink: a cluster per tile, K split over its CTAs; x and A_s stream through a ring of
// 64-wide steps into tcgen05 products that accumulate [128, R] in tensor memory, and the cluster's
// shares leave h in a scratch buffer as two bf16 parts. The expand: a tile's h stays in shared memory
// as the A operand (both parts, against the same B), y and B_s stream through a ring of 64-column units
// (gate and up: 64 of each), and the epilogue adds the product in place of y, from where whole
// 128-byte rows go out. The rows are gathered, so the ring is filled by cp.async, 16 bytes a thread. The
// tiles' units, one after another, are dealt to the resident CTAs in equal shares, which the device works
// out from the number of tiles; with runs of units from a larger grid the last CTAs ran alone (2048 rows, rank
// 64 with the epilogue, 107 against 98 us; 4096 rows, 70 % without an adapter, 30 against 27 us).
//
// It is bound by bytes, so what it takes is few instructions per byte and enough bytes in flight. 8185
// rows, K 4096, N 6144, rank up to 64 (268 MB, 42 us at the copy rate): 240 us with mma.sync fragments
// loaded from global memory, 72 us with the same behind the ring (bound by instruction issue), 60 us
// this way (4.5 TB/s). 2048 rows, K 3584, N 37888 with the epilogue (254 MB, 39 us): 151, 62, 56 to 60 us.
// A row's share of a unit is what the memory sees: 64-byte pieces gave 3.3 TB/s in the expand, 128
// bytes 4.3, 256 bytes 4.7. One CTA of 16 warps per SM instead of two of 8 was slower (66 us), with five
// stages and each product one unit ahead too (2048 rows, N 37888, rank 16, 16 adapters: 100 against 73 us):
// its phases do not overlap. Where h and the ring leave room for one CTA (rank 64 with the epilogue, rank
// 128), 16 warps are better than 8 (107 against 115 us, 70 against 75). What did not help: products one
// unit ahead beside two CTAs (8185 rows 71 against 65 us: fewer bytes in flight), wider pieces fetched to
// L2 ahead (82 against 72 us), one reciprocal for four values (80 against 73 us: longer chains).
template <int R>
struct Shrink128 {
  static constexpr int kStage = 128 * 128 + R * 128;
  static constexpr int kPart = 128 * (R + 4) * 4;  // (in the ring, once it is empty)
  static constexpr int kFit = (111 * 1024) / kStage;  // two CTAs per SM
  static constexpr int S = kFit > 5 ? 5 : kFit;
  static constexpr int kSmem = (S * kStage > kPart ? S * kStage : kPart) + 1024;
  static constexpr int kCols = R < 32 ? 32 : R;
};

template <int R>
__global__ void __launch_bounds__(kThreads, 2) lora_shrink128_kernel(const LoraParams p) {
  using TC = Shrink128<R>;
  constexpr int S = TC::S, PS = R + 4;
  static_assert(S >= 3 && TC::kStage % 1024 == 0, "ring");
  pdl_wait();
  pdl_trigger();
  if ((int)blockIdx.x >= *p.num_tiles) return;  // the whole cluster
  const int4 tile = p.tiles[blockIdx.x];
  const int slot = tile.x, cnt = tile.z;
  const int rank = slot >= 0 ? p.rank[slot] : 0;
  if (rank <= 0) return;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = align1k(smem_raw);
  float* part = reinterpret_cast<float*>(smem);  // [128][PS]
  __shared__ int rows[128];
  __shared__ __align__(8) uint64_t done[S];
  __shared__ uint32_t tmem_slot;
  cg::cluster_group cl = cg::this_cluster();
  const int C = gridDim.z, cr = blockIdx.z;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  if (tid < 128) rows[tid] = tid < cnt ? p.order[tile.y + tid] : -1;
  if (tid == 0) {
    for (int i = 0; i < S; ++i) mbar_init(&done[i], 1);
    fence_mbar_init();
  }
  if (warp == 0) {
    tmem_alloc(&tmem_slot, TC::kCols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_slot;
  const int live = min(R, (rank + 15) / 16 * 16);  // ranks computed
  const int steps = (p.K + 63) / 64;
  const int k0 = (int)((long long)steps * cr / C), n1 = (int)((long long)steps * (cr + 1) / C) - k0;

  // a thread copies chunk tid % 8 of rows tid / 8 + 32 j; the pointers run along
  const int lr = tid >> 3, lc = tid & 7;
  const __nv_bfloat16* px[4];
  unsigned on = 0;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int r = rows[lr + 32 * j];
    on |= (r >= 0 ? 1u : 0u) << j;
    px[j] = p.x + (r < 0 ? 0 : r) * p.ldx + k0 * 64 + lc * 8;
  }
  const __nv_bfloat16* pa = p.a + ((size_t)slot * R + lr) * p.K + k0 * 64 + lc * 8;
  const size_t a32 = (size_t)32 * p.K;
  const int so = sw(lr, lc);  // (rows + 32: the same swizzle)
  int kk = k0 * 64 + lc * 8, wr = 0;  // this thread's k; next stage to fill
  auto issue = [&](int i) {
    uint8_t* st = smem + wr * TC::kStage;
    wr = wr == S - 1 ? 0 : wr + 1;
    if (i < n1) {
      const bool in = kk < p.K;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        cp16(st + so + j * 4096, in ? px[j] : p.x, in && ((on >> j) & 1u));
        px[j] += 64;
      }
#pragma unroll
      for (int r = 0; r < R; r += 32)
        if (r + lr < live) cp16(st + 16384 + so + r * 128, in ? pa + (r / 32) * a32 : p.a, in);
      pa += 64;
      kk += 64;
    }
    cp_commit();
  };
#pragma unroll
  for (int i = 0; i < S - 1; ++i) issue(i);
  const uint32_t idesc = idesc_bf16_f32(128, live);
  int rd = 0;
  for (int i = 0; i < n1; ++i) {
    cp_wait<S - 2>();
    fence_proxy_async_smem();
    __syncthreads();
    if (warp == 0) {
      tc_fence_after();
      if (elect_one()) {
        const uint32_t a = smem_u32(smem + rd * TC::kStage), b = a + 16384;
#pragma unroll
        for (int k = 0; k < 4; ++k)
          mma_bf16_ss(tmem, sdesc_sw128(a + k * 32), sdesc_sw128(b + k * 32), idesc, (i > 0 || k > 0) ? 1u : 0u);
        mma_commit(&done[rd]);
      }
      __syncwarp();
    }
    // the stage to fill next is the one that the step before this one read
    if (i > 0) mbar_wait(&done[rd == 0 ? S - 1 : rd - 1], (uint32_t)((i - 1) / S) & 1u, p.status, SQ_ERR_TIMEOUT_ACC);
    issue(i + S - 1);
    rd = rd == S - 1 ? 0 : rd + 1;
  }
  if (n1 > 0) mbar_wait(&done[(n1 - 1) % S], (uint32_t)((n1 - 1) / S) & 1u, p.status, SQ_ERR_TIMEOUT_ACC);
  cp_wait<0>();
  __syncthreads();  // the ring is empty: its memory takes the shares
  tc_fence_after();
  {
    const int row = (warp & 3) * 32 + lane, c0 = (warp >> 2) * (R / 2);
    const uint32_t at = tmem + ((uint32_t)((warp & 3) * 32) << 16) + (uint32_t)c0;
    float* dst = part + row * PS + c0;
#pragma unroll
    for (int c = 0; c < R / 2; c += 8) {
      uint32_t v[8];
      tmem_ld8(at + c, v);
      tmem_wait_ld();
#pragma unroll
      for (int q = 0; q < 8; q += 4)
        *reinterpret_cast<float4*>(dst + c + q) =
            n1 > 0 ? make_float4(__uint_as_float(v[q]), __uint_as_float(v[q + 1]), __uint_as_float(v[q + 2]),
                                 __uint_as_float(v[q + 3]))
                   : make_float4(0.f, 0.f, 0.f, 0.f);
    }
    tc_fence_before();
  }
  cl.sync();
  if (warp == 0) {
    tc_fence_after();
    tmem_dealloc(tmem, TC::kCols);
  }
  // h of this CTA's share of the rows: the sum of the CTAs' shares of K, in rank order, scaled
  const float sc = p.scale[slot];
  const int r0 = 128 * cr / C, r1 = min(cnt, 128 * (cr + 1) / C);
  const int nv = live / 4;
  for (int i = tid; i < (r1 - r0) * nv; i += kThreads) {
    const int q0 = i / nv, r = r0 + q0, c = (i - q0 * nv) * 4;
    float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int q = 0; q < C; ++q) {
      const float4 v = *reinterpret_cast<const float4*>(cl.map_shared_rank(part, q) + r * PS + c);
      s.x += v.x;
      s.y += v.y;
      s.z += v.z;
      s.w += v.w;
    }
    s.x *= sc;
    s.y *= sc;
    s.z *= sc;
    s.w *= sc;
    const uint32_t h01 = pack_bf16(s.x, s.y), h23 = pack_bf16(s.z, s.w);
    __nv_bfloat16* h = p.h + (size_t)(tile.y + r) * 2 * R + c;
    *reinterpret_cast<uint2*>(h) = make_uint2(h01, h23);
    *reinterpret_cast<uint2*>(h + R) =
        make_uint2(pack_bf16(s.x - lo_f(h01), s.y - hi_f(h01)), pack_bf16(s.z - lo_f(h23), s.w - hi_f(h23)));
  }
  cl.sync();  // peers may still read this CTA's share
}

template <int R, bool SILU>
struct Expand128 {
  // 64-column halves of a unit: gate and up, or two where they fit (a row's share of a unit is then 256
  // contiguous bytes, which the memory serves faster than 128)
  static constexpr int G = SILU || R <= 32 ? 2 : 1;
  // h: [128 rows][upper | lower] in 128-byte rows; B: [64 G columns][ranks] likewise, but up to rank 32
  // the two halves share a row (64 bytes each)
  static constexpr int kA = 128 * 128 * (R >= 64 ? R / 32 : 1);
  static constexpr bool kPair = R <= 32;
  static constexpr int kBRows = kPair ? 64 : 64 * G;
  static constexpr int kB = kBRows * 128 * (R >= 64 ? R / 64 : 1);
  static constexpr int kStage = G * 128 * 128 + kB;
  static constexpr int kCtas = kA + 2 * kStage <= 111 * 1024 ? 2 : 1;  // per SM
  static constexpr int kFit = ((kCtas == 2 ? 111 : 224) * 1024 - kA) / kStage;
  static constexpr int S = kFit > 4 ? 4 : kFit;
  static constexpr int kSmem = kA + S * kStage + 1024;
  static constexpr int kCols = G * 64;
  static constexpr int T = kCtas == 2 ? 256 : 512;  // threads
};

template <int R, bool SILU>
__global__ void __launch_bounds__((Expand128<R, SILU>::T), (Expand128<R, SILU>::kCtas))
lora_expand128_kernel(const LoraParams p) {
  using TC = Expand128<R, SILU>;
  constexpr int S = TC::S, G = TC::G, T = TC::T;
  constexpr int RP = T / 8, RJ = 128 / RP;  // rows per pass of the block's copies, passes
  constexpr int OQ = SILU ? 1 : G;  // 64-column halves of the output of a unit
  static_assert(S >= 2 && TC::kStage % 1024 == 0, "ring");
  // The launch before this one is the shrink, which lets this one start once everything before it is
  // complete: the plan, y and B may be read at once, h after the wait.
  const int units = (p.N + 64 * G - 1) / (64 * G);
  int nt = *p.num_tiles;
  // in place, the rows without an adapter (the last tiles) are left as they are: no CTA's share holds them
  if (p.in_place) {
    int n = 0;
    for (int i = threadIdx.x; i < nt; i += T) n += p.tiles[i].x >= 0;
    __shared__ int with;
    if (threadIdx.x == 0) with = 0;
    __syncthreads();
    n = __reduce_add_sync(0xffffffffu, n);
    if ((threadIdx.x & 31) == 0) atomicAdd(&with, n);
    __syncthreads();
    nt = with;
  }
  const long long total = (long long)nt * units;
  long long at0 = total * blockIdx.x / gridDim.x;
  const long long at1 = total * (blockIdx.x + 1) / gridDim.x;
  if (at0 >= at1) {
    pdl_wait();
    pdl_trigger();
    return;
  }
  extern __shared__ uint8_t smem_raw[];
  uint8_t* ha = align1k(smem_raw);
  uint8_t* ring = ha + TC::kA;
  __shared__ int rows[128];
  __shared__ __align__(8) uint64_t done;
  __shared__ uint32_t tmem_slot;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  if (tid == 0) {
    mbar_init(&done, 1);
    fence_mbar_init();
  }
  if (warp == 0) {
    tmem_alloc(&tmem_slot, TC::kCols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_slot;
  bool waited = false;
  uint32_t phase = 0;  // of the next product

  while (at0 < at1) {  // a tile's part of this CTA's share: units u0 .. u0 + n2
    const int ti = (int)(at0 / units);
    const int u0 = (int)(at0 - (long long)ti * units), n2 = (int)min((long long)(units - u0), at1 - at0);
    at0 += n2;
    const int4 tile = p.tiles[ti];
    const int slot = tile.x, cnt = tile.z;
    const int rank = slot >= 0 ? p.rank[slot] : 0;
    if (rank <= 0 && p.in_place) continue;
    const int live = rank <= 0 ? 0 : min(R, (rank + 15) / 16 * 16);
    if (tid < 128) rows[tid] = tid < cnt ? p.order[tile.y + tid] : -1;
    __syncthreads();

    // a thread copies chunk tid % 8 of rows tid / 8 + RP j of y (and of out), and pieces of B rows
    const int lr = tid >> 3, lc = tid & 7;
    const __nv_bfloat16* py[RJ];
    __nv_bfloat16* po[RJ];
    unsigned on = 0;
#pragma unroll
    for (int j = 0; j < RJ; ++j) {
      const int r = rows[lr + RP * j];
      on |= (r >= 0 ? 1u : 0u) << j;
      py[j] = p.y + (r < 0 ? 0 : r) * p.ldy + (long long)u0 * 64 * G + lc * 8;
      po[j] = p.out + (r < 0 ? 0 : r) * p.ldo + (long long)u0 * 64 * OQ + lc * 8;
    }
    constexpr int CH = R / 8;          // 16-byte pieces of a B row
    constexpr int BN = T / CH;         // B rows per pass
    const int bn = tid / CH, bc = tid % CH;
    const __nv_bfloat16* pb = p.b + ((size_t)(slot < 0 ? 0 : slot) * p.N + (size_t)u0 * 64 * G + bn) * R + bc * 8;
    const int so = sw(lr, lc);
    int col = u0 * 64 * G, wr = 0;  // the unit's first column; next stage to fill
    auto issue = [&](int i) {
      uint8_t* st = ring + wr * TC::kStage;
      wr = wr == S - 1 ? 0 : wr + 1;
      if (i < n2) {
#pragma unroll
        for (int j = 0; j < RJ; ++j) {
#pragma unroll
          for (int q = 0; q < G; ++q) {
            const bool in = SILU || col + q * 64 + lc * 8 < p.N;
            cp16(st + q * 16384 + so + j * RP * 128, in ? py[j] + q * 64 : p.y, in && ((on >> j) & 1u));
          }
          py[j] += 64 * G;
        }
        if (bc * 8 < live) {
#pragma unroll
          for (int k = 0; k < G * 64; k += BN) {
            const int n = bn + k;
            if (BN > G * 64 && n >= G * 64) break;
            const bool ok = SILU || col + n < p.N;
            const int at = TC::kPair ? sw(n & 63, (n >> 6) * 4 + bc) : (bc >> 3) * (G * 8192) + sw(n, bc & 7);
            cp16(st + G * 16384 + at, ok ? pb + (size_t)k * R : p.b, ok);
          }
        }
        pb += (size_t)64 * G * R;
        col += 64 * G;
      }
      cp_commit();
    };
#pragma unroll
    for (int i = 0; i < S - 1; ++i) issue(i);
    if (!waited) {
      pdl_wait();
      pdl_trigger();
      waited = true;
    }
    if (live > 0) {  // h of the tile, as the A operand
      for (int e = tid; e < 128 * 2 * CH; e += T) {
        const int r = e / (2 * CH), q = e / CH % 2, c = e % CH;
        if (c * 8 < live) {
          const int at = R >= 64 ? (q * (R / 64) + (c >> 3)) * 16384 + sw(r, c & 7) : sw(r, q * CH + c);
          cp16(ha + at, r < cnt ? p.h + ((size_t)(tile.y + r) * 2 + q) * R + c * 8 : p.h, r < cnt);
        }
      }
    }
    cp_commit();
    constexpr int TQ = 8192 / T;                             // columns of a half per thread
    const int row = (warp & 3) * 32 + lane, hf = warp >> 2;  // this thread's row and part of the columns
    const uint32_t lanes = tmem + ((uint32_t)((warp & 3) * 32) << 16);
    constexpr uint32_t idesc = idesc_bf16_f32(128, TC::kPair ? 64 : 64 * G);
    int rd = 0;
    for (int i = 0; i < n2; ++i) {
      if (i == 0) cp_wait<0>();
      else cp_wait<S - 2>();
      fence_proxy_async_smem();
      __syncthreads();
      uint8_t* st = ring + rd * TC::kStage;
      rd = rd == S - 1 ? 0 : rd + 1;
      if (live > 0 && warp == 0) {
        tc_fence_after();
        if (elect_one()) {
          const uint32_t a = smem_u32(ha), b = smem_u32(st + G * 16384);
#pragma unroll
          for (int g = 0; g < (TC::kPair ? 2 : 1); ++g)  // (gate, up)
#pragma unroll
            for (int q = 1; q >= 0; --q)  // lower part first
              for (int ks = 0; ks < live / 16; ++ks) {
                const uint32_t ao = R >= 64 ? (q * (R / 64) + (ks >> 2)) * 16384 + (ks & 3) * 32 : (q * R / 16 + ks) * 32;
                const uint32_t bo = TC::kPair ? g * 64 + ks * 32 : (ks >> 2) * (G * 8192) + (ks & 3) * 32;
                mma_bf16_ss(tmem + g * 64, sdesc_sw128(a + ao), sdesc_sw128(b + bo), idesc, q == 0 || ks > 0 ? 1u : 0u);
              }
          mma_commit(&done);
        }
        __syncwarp();
      }
      issue(i + S - 1);  // (its stage was emptied by the step before this one)
      if (live > 0) {
        mbar_wait(&done, phase, p.status, SQ_ERR_TIMEOUT_ACC);
        phase ^= 1u;
        tc_fence_after();
      }
      // the thread's output columns of each half of its row, in place of y
#pragma unroll
      for (int oq = 0; oq < OQ; ++oq) {
        uint32_t vs[TQ / 16][2][16];  // products (SiLU*up: of the gate and of the up columns)
        if (live > 0) {
#pragma unroll
          for (int c = 0; c < TQ / 16; ++c) {
            tmem_ld16(lanes + oq * 64 + hf * TQ + c * 16, vs[c][0]);
            if (SILU) tmem_ld16(lanes + 64 + hf * TQ + c * 16, vs[c][1]);
          }
          tmem_wait_ld();
        } else {
#pragma unroll
          for (int c = 0; c < TQ / 16; ++c)
#pragma unroll
            for (int k = 0; k < 16; ++k) vs[c][0][k] = vs[c][1][k] = 0u;
        }
#pragma unroll
        for (int c = 0; c < TQ; c += 16) {
          const int c0 = hf * TQ + c;
          auto& v = vs[c / 16];
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            uint4* at = reinterpret_cast<uint4*>(st + oq * 16384 + sw(row, c0 / 8 + h));
            const uint4 y = *at;
            const uint32_t yw[4] = {y.x, y.y, y.z, y.w};
            uint32_t uw[4] = {0, 0, 0, 0};
            if (SILU) {
              const uint4 x = *reinterpret_cast<const uint4*>(st + 16384 + sw(row, c0 / 8 + h));
              uw[0] = x.x;
              uw[1] = x.y;
              uw[2] = x.z;
              uw[3] = x.w;
            }
            uint32_t o[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              float f0 = lo_f(yw[k]) + __uint_as_float(v[0][8 * h + 2 * k]);
              float f1 = hi_f(yw[k]) + __uint_as_float(v[0][8 * h + 2 * k + 1]);
              if (SILU) {
                f0 = silu_mul(f0, lo_f(uw[k]) + __uint_as_float(v[1][8 * h + 2 * k]));
                f1 = silu_mul(f1, hi_f(uw[k]) + __uint_as_float(v[1][8 * h + 2 * k + 1]));
              }
              o[k] = pack_bf16(f0, f1);
            }
            *at = make_uint4(o[0], o[1], o[2], o[3]);
          }
        }
      }
      tc_fence_before();
      __syncthreads();
#pragma unroll
      for (int j = 0; j < RJ; ++j) {
#pragma unroll
        for (int oq = 0; oq < OQ; ++oq)
          if (((on >> j) & 1u) && (SILU || (u0 + i) * 64 * OQ + oq * 64 + lc * 8 < p.N))
            *reinterpret_cast<uint4*>(po[j] + oq * 64) = *reinterpret_cast<const uint4*>(st + oq * 16384 + so + j * RP * 128);
        po[j] += 64 * OQ;
      }
    }
    cp_wait<0>();
    __syncthreads();
  }
  if (!waited) {
    pdl_wait();
    pdl_trigger();
  }
  if (warp == 0) {
    tc_fence_after();
    tmem_dealloc(tmem, TC::kCols);
  }
}

template <int R, bool SILU>
cudaError_t launch_lora(const LoraParams& p, int C, int num_sms, cudaStream_t s) {
  if (p.tm == 16) {
    constexpr size_t smem = (size_t)kWarps * 16 * (R + 4) * 4 + (size_t)2 * 16 * (R + 8) * 2;
    if (smem > 48 * 1024) {
      const cudaError_t e = allow_smem(lora_row16_kernel<R, SILU>, (int)smem);
      if (e != cudaSuccess) return e;
    }
    // Clusters per tile: few tiles and many columns leave SMs idle, so up to 8 clusters share a tile's
    // columns, each computing h again (A comes from L2), while a warp keeps two units or more. Measured
    // with 1, 2, 4, 8: 1 row, N 37888 with the epilogue 13.9, 9.2, 7.3, 6.6 us; 64 rows over 16 adapters
    // 16.6, 13.7, 18.2, 22.9 us; 64 rows over 32 adapters, N 4608 7.0, 8.9, 14.4, 23.7 us.
    const int units = SILU ? p.N / 64 : (p.N + 31) / 32;
    int split = 1;
    while (split < 8 && p.max_tiles * C * split * 2 <= 4 * num_sms && units >= C * kWarps * 2 * split * 2) split *= 2;
    SQ_LAUNCH((lora_row16_kernel<R, SILU>), dim3(p.max_tiles, split, C), dim3(kThreads), smem, s, C, p);
    return cudaGetLastError();
  }
  cudaError_t e = allow_smem(lora_shrink128_kernel<R>, Shrink128<R>::kSmem);
  if (e != cudaSuccess) return e;
  SQ_LAUNCH(lora_shrink128_kernel<R>, dim3(p.max_tiles, 1, C), dim3(kThreads), (size_t)Shrink128<R>::kSmem, s, C, p);
  using TC = Expand128<R, SILU>;
  e = allow_smem(lora_expand128_kernel<R, SILU>, TC::kSmem);
  if (e != cudaSuccess) return e;
  // the tiles' units in equal shares
  const int units = (p.N + 64 * TC::G - 1) / (64 * TC::G);
  const long long work = (long long)p.max_tiles * units;
  const int ctas = (int)(work < 2ll * TC::kCtas * num_sms ? (work + 1) / 2 : TC::kCtas * num_sms);
  SQ_LAUNCH((lora_expand128_kernel<R, SILU>), dim3(ctas), dim3(TC::T), (size_t)TC::kSmem, s, 1, p);
  return cudaGetLastError();
}

template <int R>
cudaError_t launch_rank(const LoraParams& p, int C, int num_sms, cudaStream_t s) {
  return p.silu ? launch_lora<R, true>(p, C, num_sms, s) : launch_lora<R, false>(p, C, num_sms, s);
}

}  // namespace

cudaError_t lora_plan_launch(const LoraPlanParams& p, cudaStream_t s) {
  if (p.slots < 1 || p.slots > kLoraMaxSlots || (p.tm != 16 && p.tm != 128)) return cudaErrorInvalidValue;
  const size_t smem = (size_t)(kPlanWarps * (p.slots + 1) + 2 * (p.slots + 2)) * sizeof(int);
  if (smem > 48 * 1024) {
    const cudaError_t e = allow_smem(lora_plan_kernel, (kPlanWarps * (kLoraMaxSlots + 1) + 2 * (kLoraMaxSlots + 2)) * 4);
    if (e != cudaSuccess) return e;
  }
  SQ_LAUNCH(lora_plan_kernel, dim3(1), dim3(kPlanThreads), smem, s, 1, p);
  return cudaGetLastError();
}

cudaError_t lora_add_launch(const LoraParams& p, int num_sms, cudaStream_t s) {
  if (p.M == 0 || p.N == 0) return cudaSuccess;
  if (p.K % 8 || p.N % 8 || (p.silu && p.N % 128) || (p.tm != 16 && p.tm != 128)) return cudaErrorInvalidValue;
  // CTAs per tile (K split over them): more while few tiles leave SMs idle. Measured with 2, 4, 8, tiles
  // of 128 rows: 33 tiles at most, K 3584: 64, 60, 58 us; 82 tiles, K 4096: 65, 61, 65 us; 72 tiles, K
  // 2048: 40, 38, 45 us. Tiles of 16 rows: 1 row 9.4, 7.1, 6.0 us; 37 tiles at most 10.5, 8.0, 8.0 us.
  // (The number of tiles is known on the device only; its bound grows with the pool's slots, so a large
  // pool of which a step uses a few gets fewer CTAs than it could: see ops.LoraPool for what that costs.)
  int C = 8;
  while (C > 1 && p.max_tiles * C > (p.tm == 16 ? 4 : 3) * num_sms) C >>= 1;
  switch (p.R) {
    case 16: return launch_rank<16>(p, C, num_sms, s);
    case 32: return launch_rank<32>(p, C, num_sms, s);
    case 64: return launch_rank<64>(p, C, num_sms, s);
    case 128: return launch_rank<128>(p, C, num_sms, s);
    default: return cudaErrorInvalidValue;
  }
}

}  // namespace sq
