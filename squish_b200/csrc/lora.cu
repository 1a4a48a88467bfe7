// lora.cu — low-rank adapters of many requests at once beside a shared projection.
//
//   out[t] = y[t] + scale[s] * B_s (A_s x[t])       s = adapter slot of row t (none: out[t] = y[t])
// optionally followed by the SiLU(gate) * up epilogue over [gate 64 | up 64] column blocks.
//
// The plan (lora_plan, once per step, shared by every projection) sorts the rows by slot, stable, and
// cuts them into tiles of at most tm rows of one adapter. One cluster of C CTAs computes a tile in one
// launch: each CTA takes 1/C of K and computes its share of h = A_s x (tm x R) on the tensor cores,
// the shares meet through the cluster's shared memory in fp32, and each CTA then takes 1/C of the
// output columns. x, y and out cross HBM once; h never leaves the cluster.
//
// The work is bound by bytes (y and out dominate): per row and projection 2 r (K + N) flops against
// 2 (K + 2 N) bytes. Operands go straight from global memory into mma fragments: the order of k
// within a 32-value step is free as long as both operands agree, so a lane takes 8 consecutive
// values (16 bytes) of its row, and the columns of four 8-wide tiles are interleaved so that a lane's
// accumulators are 8 consecutive columns of out (16-byte loads of y, 16-byte stores of out).
//
// h is held in fp32 and enters the second product as a sum of two bf16 (upper and lower part, 16
// bits of h): out is rounded once, as the formula would be; one bf16 alone would add an error of
// 2^-9 |h| per rank to every column. The rank is small, so the second product costs no time.
#include <cooperative_groups.h>

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
// y added to the accumulators of 16 rows x 32 columns: a lane's 8 columns of its two rows ...
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
// ... or as their start, where y is at hand before the products (16 additions and 16 zeros fewer).
__device__ __forceinline__ void start_from(float (&acc)[4][4], uint4 y0, uint4 y1) {
  const uint32_t w0[4] = {y0.x, y0.y, y0.z, y0.w}, w1[4] = {y1.x, y1.y, y1.z, y1.w};
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const uint32_t a = w0[j], b = w1[j];
    acc[j][0] = lo_f(a);
    acc[j][1] = hi_f(a);
    acc[j][2] = lo_f(b);
    acc[j][3] = hi_f(b);
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

// Tiles of 16 rows (decode). R: padded rank of the pool.
template <int R, bool SILU>
__global__ void __launch_bounds__(kThreads) lora_row16_kernel(const LoraParams p) {
  constexpr int RT = R / 8;           // 8-wide rank tiles
  constexpr int KW = kWarps;          // the warps split K (shrink), then the columns (expand)
  constexpr int ROWS = 16;
  constexpr int PS = R + 4;           // row stride of the fp32 shares (4: rows on distinct banks)
  constexpr int HS = R + 8;           // row stride of the bf16 parts of h
  pdl_wait();
  pdl_trigger();
  if ((int)blockIdx.x >= *p.num_tiles) return;  // the whole cluster
  const int4 tile = p.tiles[blockIdx.x];
  const int slot = tile.x, cnt = tile.z;
  const int rank = slot >= 0 ? p.rank[slot] : 0;
  if (rank <= 0 && p.in_place) return;
  extern __shared__ __align__(16) uint8_t smem[];
  float* part = reinterpret_cast<float*>(smem);                                    // [KW][ROWS][PS]
  __nv_bfloat16* hh = reinterpret_cast<__nv_bfloat16*>(part + KW * ROWS * PS);     // [2][ROWS][HS]
  __shared__ int rows[ROWS];
  cg::cluster_group cl = cg::this_cluster();
  const int C = gridDim.z, cr = blockIdx.z;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int g = lane >> 2, t = lane & 3;
  const int kw = warp;
  if (tid < ROWS) rows[tid] = tid < cnt ? p.order[tile.y + tid] : -1;
  __syncthreads();
  const int row0 = rows[g], row1 = rows[g + 8];
  const int live = min(R, (rank + 15) / 16 * 16);  // ranks computed: whole 16-wide steps

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
    const float sc = p.scale[slot];
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
    __syncthreads();
  }

  // ---- out = y + h B^T over this CTA's columns, 32 output columns per step
  constexpr int KS = R == 16 ? 1 : R / 32;  // rank steps (32 wide; one of 16 for R = 16)
  constexpr int G = SILU ? 2 : 1;           // column groups of a step (gate and up)
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
  const __nv_bfloat16* bs = p.b + (size_t)(slot < 0 ? 0 : slot) * p.N * R;
  const int units = SILU ? p.N / 64 : (p.N + 31) / 32;
  const int u0 = (int)((long long)units * cr / C), u1 = (int)((long long)units * (cr + 1) / C);
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
  if (rank > 0) cl.sync();  // peers may still read this CTA's share
}

// ---------------------------------------------------------------- tiles of 64 rows (prefill)
__device__ __forceinline__ void cp16(void* dst, const void* src, bool on) {  // 16 bytes, or zeros
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(dst)), "l"(src), "r"(on ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
// Offset of 16-byte chunk c (0..7) of row r in a tile of 128-byte rows. A fragment load reads four
// chunks of two neighbouring rows per phase: odd rows swap their halves, so they meet no bank twice.
__device__ __forceinline__ int sw(int r, int c) { return r * 128 + ((c ^ ((r & 1) << 2)) << 4); }

// 8 warps: 4 row groups of 16 x 2 halves (of the rank tiles in the shrink, of the columns in the
// expand). One ring of stages runs through both products: x and A in 64-wide steps of K, then y and
// B in units of 64 columns (gate and up: 128), so the first units of y are in flight while the
// cluster exchanges h. The loads are what bounds it: without the ring each warp waited for its own
// fragments (8185 rows, K 4096, N 6144, rank 64: 240 us, 1.1 TB/s).
template <int R, bool SILU>
struct Tile64 {
  static constexpr int G = SILU ? 2 : 1;
  static constexpr int kStage = G * 64 * 128 + G * 64 * R * 2 > 64 * 128 + R * 128 ? G * 64 * 128 + G * 64 * R * 2
                                                                                  : 64 * 128 + R * 128;
  static constexpr int kPart = 64 * (R + 4) * 4, kH = 2 * 64 * (R + 8) * 2;
  // as many stages as two resident CTAs leave room for, at least two
  static constexpr int kFit = (113 * 1024 - kPart - kH - 1024) / kStage;
  static constexpr int S = kFit > 5 ? 5 : kFit < 2 ? 2 : kFit;
  static constexpr int kSmem = S * kStage + kPart + kH;
};

template <int R, bool SILU>
__global__ void __launch_bounds__(kThreads) lora_row64_kernel(const LoraParams p) {
  using TC = Tile64<R, SILU>;
  constexpr int S = TC::S, G = TC::G;
  constexpr int RH = R / 16;        // 8-wide rank tiles of a warp: 2 i + half
  constexpr int PS = R + 4, HS = R + 8;
  pdl_wait();
  pdl_trigger();
  if ((int)blockIdx.x >= *p.num_tiles) return;  // the whole cluster
  const int4 tile = p.tiles[blockIdx.x];
  const int slot = tile.x, cnt = tile.z;
  const int rank = slot >= 0 ? p.rank[slot] : 0;
  if (rank <= 0 && p.in_place) return;
  extern __shared__ __align__(128) uint8_t smem[];
  float* part = reinterpret_cast<float*>(smem + S * TC::kStage);                         // [64][PS]
  __nv_bfloat16* hh = reinterpret_cast<__nv_bfloat16*>(smem + S * TC::kStage + TC::kPart);  // [2][64][HS]
  __shared__ int rows[64];
  cg::cluster_group cl = cg::this_cluster();
  const int C = gridDim.z, cr = blockIdx.z;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int g = lane >> 2, t = lane & 3;
  const int rw = warp >> 1, hf = warp & 1;
  if (tid < 64) rows[tid] = tid < cnt ? p.order[tile.y + tid] : -1;
  __syncthreads();
  const int live = min(R, (rank + 15) / 16 * 16);
  const int steps = rank > 0 ? (p.K + 63) / 64 : 0;
  const int k0 = (int)((long long)steps * cr / C), n1 = (int)((long long)steps * (cr + 1) / C) - k0;
  const int units = (p.N + 64 * G - 1) / (64 * G);
  const int u0 = (int)((long long)units * cr / C), n2 = (int)((long long)units * (cr + 1) / C) - u0;
  const __nv_bfloat16* as = p.a + (size_t)(slot < 0 ? 0 : slot) * R * p.K;
  const __nv_bfloat16* bs = p.b + (size_t)(slot < 0 ? 0 : slot) * p.N * R;

  // a thread copies chunk tid % 8 of rows tid / 8 and tid / 8 + 32 of a 64-row tile
  const int lr = tid >> 3, lc = tid & 7;
  const int ra = rows[lr], rb = rows[lr + 32];
  const __nv_bfloat16* xa = p.x + (ra < 0 ? 0 : ra) * p.ldx + lc * 8;
  const __nv_bfloat16* xb = p.x + (rb < 0 ? 0 : rb) * p.ldx + lc * 8;
  const __nv_bfloat16* ya = p.y + (ra < 0 ? 0 : ra) * p.ldy + lc * 8;
  const __nv_bfloat16* yb = p.y + (rb < 0 ? 0 : rb) * p.ldy + lc * 8;
  int wr = 0, rd = 0;  // offsets of the next stage to fill and to use
  auto next = [](int& at) { at = at == (S - 1) * TC::kStage ? 0 : at + TC::kStage; };
  auto issue = [&](int i) {
    uint8_t* st = smem + wr;
    next(wr);
    if (i < n1) {
      const int k = (k0 + i) * 64;
      const bool in = k + lc * 8 < p.K;
      cp16(st + sw(lr, lc), in ? xa + k : p.x, in && ra >= 0);
      cp16(st + sw(lr + 32, lc), in ? xb + k : p.x, in && rb >= 0);
      uint8_t* sa = st + 64 * 128;
#pragma unroll
      for (int r = 0; r < R; r += 32)
        if (r + lr < live) cp16(sa + sw(r + lr, lc), in ? as + (size_t)(r + lr) * p.K + k + lc * 8 : as, in);
    } else if (i < n1 + n2) {
      const int col = (u0 + i - n1) * 64 * G;
#pragma unroll
      for (int q = 0; q < G; ++q) {
        const int c = col + q * 64;
        const bool in = c + lc * 8 < p.N;
        cp16(st + q * 8192 + sw(lr, lc), in ? ya + c : p.y, in && ra >= 0);
        cp16(st + q * 8192 + sw(lr + 32, lc), in ? yb + c : p.y, in && rb >= 0);
      }
      uint8_t* sb = st + G * 8192;
      constexpr int CH = R / 8;  // 16-byte pieces of a B row
      const int c = tid % CH;
      if (c * 8 < live) {
#pragma unroll
        for (int n = tid / CH; n < G * 64; n += kThreads / CH) {
          const bool in = col + n < p.N;
          const __nv_bfloat16* src = in ? bs + (size_t)(col + n) * R + c * 8 : bs;
          if (R >= 64) cp16(sb + (c >> 3) * (G * 64 * 128) + sw(n, c & 7), src, in);
          else cp16(sb + n * R * 2 + c * 16, src, in);
        }
      }
    }
    cp_commit();
  };
#pragma unroll
  for (int i = 0; i < S - 1; ++i) issue(i);

  // ---- shrink
  if (rank > 0) {
    float acc[RH][4];
#pragma unroll
    for (int i = 0; i < RH; ++i) acc[i][0] = acc[i][1] = acc[i][2] = acc[i][3] = 0.f;
    for (int i = 0; i < n1; ++i) {
      cp_wait<S - 2>();
      __syncthreads();
      issue(i + S - 1);
      const uint8_t* st = smem + rd;
      next(rd);
      const uint8_t* sa = st + 64 * 128;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const uint4 v0 = *reinterpret_cast<const uint4*>(st + sw(rw * 16 + g, h * 4 + t));
        const uint4 v1 = *reinterpret_cast<const uint4*>(st + sw(rw * 16 + g + 8, h * 4 + t));
        uint4 w[RH];
#pragma unroll
        for (int j = 0; j < RH; ++j)
          if ((2 * j + hf) * 8 < live) w[j] = *reinterpret_cast<const uint4*>(sa + sw((2 * j + hf) * 8 + g, h * 4 + t));
#pragma unroll
        for (int j = 0; j < RH; ++j)
          if ((2 * j + hf) * 8 < live) mma16816(acc[j], v0.x, v1.x, v0.y, v1.y, w[j].x, w[j].y);
#pragma unroll
        for (int j = 0; j < RH; ++j)
          if ((2 * j + hf) * 8 < live) mma16816(acc[j], v0.z, v1.z, v0.w, v1.w, w[j].z, w[j].w);
      }
    }
#pragma unroll
    for (int j = 0; j < RH; ++j) {
      const int c = (2 * j + hf) * 8 + 2 * t;
      if ((2 * j + hf) * 8 >= live) break;
      *reinterpret_cast<float2*>(part + (rw * 16 + g) * PS + c) = make_float2(acc[j][0], acc[j][1]);
      *reinterpret_cast<float2*>(part + (rw * 16 + g + 8) * PS + c) = make_float2(acc[j][2], acc[j][3]);
    }
    cl.sync();
    const float sc = p.scale[slot];
    const int nv = live / 4;
    for (int i = tid; i < 64 * nv; i += kThreads) {
      const int r = i / nv, c = (i - r * nv) * 4;
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
      *reinterpret_cast<uint2*>(hh + r * HS + c) = make_uint2(h01, h23);
      *reinterpret_cast<uint2*>(hh + (64 + r) * HS + c) =
          make_uint2(pack_bf16(s.x - lo_f(h01), s.y - hi_f(h01)), pack_bf16(s.z - lo_f(h23), s.w - hi_f(h23)));
    }
    __syncthreads();
  }

  // ---- expand
  constexpr int KS = R == 16 ? 1 : R / 32;
  uint4 fa[2][KS][2];
#pragma unroll
  for (int q = 0; q < 2; ++q)
#pragma unroll
    for (int ks = 0; ks < KS; ++ks)
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const __nv_bfloat16* src = hh + (q * 64 + rw * 16 + g + 8 * r) * HS;
        fa[q][ks][r] = make_uint4(0, 0, 0, 0);
        if (R == 16) {
          if (rank > 0) {
            const uint2 v = *reinterpret_cast<const uint2*>(src + t * 4);
            fa[q][ks][r].x = v.x;
            fa[q][ks][r].y = v.y;
          }
        } else if (ks * 32 + t * 8 < live) {
          fa[q][ks][r] = *reinterpret_cast<const uint4*>(src + ks * 32 + t * 8);
        }
      }
  const int row0 = rows[rw * 16 + g], row1 = rows[rw * 16 + g + 8];
  for (int i = n1; i < n1 + n2; ++i) {
    cp_wait<S - 2>();
    __syncthreads();
    issue(i + S - 1);
    const uint8_t* st = smem + rd;
    next(rd);
    const uint8_t* sb = st + G * 8192;
    float acc[G][4][4];
#pragma unroll
    for (int q = 0; q < G; ++q) {
      start_from(acc[q], *reinterpret_cast<const uint4*>(st + q * 8192 + sw(rw * 16 + g, hf * 4 + t)),
                 *reinterpret_cast<const uint4*>(st + q * 8192 + sw(rw * 16 + g + 8, hf * 4 + t)));
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        if (ks * 32 >= live) break;
        uint4 w[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int n = q * 64 + hf * 32 + (g >> 1) * 8 + 2 * j + (g & 1);
          w[j] = make_uint4(0, 0, 0, 0);
          if (R == 16) {
            const uint2 v = *reinterpret_cast<const uint2*>(sb + n * R * 2 + t * 8);
            w[j].x = v.x;
            w[j].y = v.y;
          } else if (ks * 32 + t * 8 < live) {
            if (R >= 64) w[j] = *reinterpret_cast<const uint4*>(sb + (ks >> 1) * (G * 64 * 128) + sw(n, (ks & 1) * 4 + t));
            else w[j] = *reinterpret_cast<const uint4*>(sb + n * R * 2 + t * 16);
          }
        }
        expand_step<R>(acc[q], fa[1][ks], fa[0][ks], w);
      }
    }
    const int oc = (u0 + i - n1) * 64 + hf * 32 + t * 8;
    if (SILU || oc < p.N) {
      if (row0 >= 0) *reinterpret_cast<uint4*>(p.out + row0 * p.ldo + oc) = finish<SILU, G>(acc, 0);
      if (row1 >= 0) *reinterpret_cast<uint4*>(p.out + row1 * p.ldo + oc) = finish<SILU, G>(acc, 1);
    }
  }
  if (rank > 0) cl.sync();  // peers may still read this CTA's share
}

template <int R, bool SILU>
cudaError_t launch_lora(const LoraParams& p, int C, cudaStream_t s) {
  const bool small = p.tm == 16;
  constexpr size_t smem16 = (size_t)kWarps * 16 * (R + 4) * 4 + (size_t)2 * 16 * (R + 8) * 2;
  const size_t smem = small ? smem16 : (size_t)Tile64<R, SILU>::kSmem;
  auto* kern = small ? lora_row16_kernel<R, SILU> : lora_row64_kernel<R, SILU>;
  if (smem > 48 * 1024) {
    const cudaError_t e = allow_smem(kern, (int)smem);
    if (e != cudaSuccess) return e;
  }
  SQ_LAUNCH(kern, dim3(p.max_tiles, 1, C), dim3(kThreads), smem, s, C, p);
  return cudaGetLastError();
}

template <int R>
cudaError_t launch_rank(const LoraParams& p, int C, cudaStream_t s) {
  return p.silu ? launch_lora<R, true>(p, C, s) : launch_lora<R, false>(p, C, s);
}

}  // namespace

cudaError_t lora_plan_launch(const LoraPlanParams& p, cudaStream_t s) {
  if (p.slots < 1 || p.slots > kLoraMaxSlots || (p.tm != 16 && p.tm != 64)) return cudaErrorInvalidValue;
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
  if (p.K % 8 || p.N % 8 || (p.silu && p.N % 128) || (p.tm != 16 && p.tm != 64)) return cudaErrorInvalidValue;
  int C = 8;
  while (C > 1 && p.max_tiles * C > 4 * num_sms) C >>= 1;
  switch (p.R) {
    case 16: return launch_rank<16>(p, C, s);
    case 32: return launch_rank<32>(p, C, s);
    case 64: return launch_rank<64>(p, C, s);
    case 128: return launch_rank<128>(p, C, s);
    default: return cudaErrorInvalidValue;
  }
}

}  // namespace sq
