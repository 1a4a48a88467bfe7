// step_ops.h — launch interfaces of the serving-step operators: the step's layout (block tables,
// slot map, attention tiles), low-rank adapters of many requests, scored expert routing and
// sampling from given uniform numbers.
#pragma once
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <cstdint>

namespace sq {

// Dynamic shared memory above 48 KB has to be allowed once per kernel and device (a driver call of its
// own: not one per launch). Kernels without a size that varies call it with their largest.
template <typename K>
cudaError_t allow_smem(K* kernel, int bytes) {
  struct Done {
    const void* kernel;
    int device;
  };
  static thread_local Done done[64];
  static thread_local int n = 0;
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  const void* k = reinterpret_cast<const void*>(kernel);
  for (int i = 0; i < n; ++i)
    if (done[i].kernel == k && done[i].device == dev) return cudaSuccess;
  e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e == cudaSuccess && n < 64) done[n++] = {k, dev};
  return e;
}

// ---------------------------------------------------------------- step layout (step_layout.cu)
constexpr int kLayoutMaxSeqs = 8192;       // per-sequence prefixes live in shared memory (16 B each)
constexpr int kLayoutPadQ0 = 1 << 30;      // first query of a padding tile: past every chunk's end
struct StepLayoutParams {
  const int* ctx_len;     // [B] tokens already in the cache
  const int* q_len;       // [B] tokens of this step
  int* block_tables;      // [B, bt_stride]; the first ceil(ctx / page) entries of a row are its pages
  int bt_stride, bt_width;
  const int* free_pages;  // [n_free] pages handed out in sequence order, from the front
  int n_free;
  int B, page_size, tile, token_cap, tile_cap;
  int* q_start;    // [B + 1]
  int* kv_len;     // [B]
  int* positions;  // [token_cap], like the next two 16-byte aligned and padded to a multiple of 4
  int* slots;      // [token_cap]
  int* token_seq;  // [token_cap]
  int* last_row;   // [B]
  int* tile_seq;   // [tile_cap]
  int* tile_q0;    // [tile_cap]
  int* totals;     // [3] tokens, new pages, tiles
  int* status;
};
cudaError_t step_layout_launch(const StepLayoutParams& p, int num_sms, cudaStream_t s);

// ---------------------------------------------------------------- scored routing (moe_scored.cu)
constexpr int kRouteMaxExperts = 512, kRouteMaxGroups = 32, kRouteMaxK = 32;
struct RouteScoredParams {
  const void* logits;  // [T, ld] bf16 or fp32
  int ld, T, E, K;
  bool f32;
  bool sigmoid;        // else softmax over the E logits
  const float* bias;   // [E] added for the choice only, or nullptr
  int groups, top_groups;
  bool top2;           // group score: sum of its two best choice scores (else its best)
  bool renorm;
  float scale;
  int* ids;    // [T * K]
  float* w;    // [T * K]
};
cudaError_t moe_route_scored_launch(const RouteScoredParams& p, cudaStream_t s);

// ---------------------------------------------------------------- sampling (sample_uniform.cu)
struct SampleUniformParams {
  const __nv_bfloat16* logits;  // [B, ld]
  long long ld;
  int V, B;
  const float* uniforms;        // [B] in [0, 1)
  const float* temperature;     // [B] (<= 0 -> greedy) or nullptr (greedy)
  const float* top_p;           // [B] (>= 1 -> off) or nullptr
  const int* top_k;             // [B] (<= 0 -> off) or nullptr
  const float* min_p;           // [B] (<= 0 -> off) or nullptr
  const uint32_t* allow_mask;   // [B, ceil(V / 32)] or nullptr
  int* out_tokens;              // [B]
  float* out_logprob;           // [B] or nullptr
};
cudaError_t sample_uniform_launch(const SampleUniformParams& p, int num_sms, cudaStream_t s);

// ---------------------------------------------------------------- adapters (lora.cu)
constexpr int kLoraMaxSlots = 1024, kLoraMaxRank = 128;
struct LoraPlanParams {
  const int* row_slot;  // [M] adapter slot of each row, -1 = none
  int M, slots, tm;
  int* order;      // [M] rows sorted by slot (stable), rows without an adapter last
  int4* tiles;     // [max_tiles] (slot or -1, first position in order, rows, 0)
  int max_tiles;
  int* num_tiles;  // [1]
  int* status;
};
cudaError_t lora_plan_launch(const LoraPlanParams& p, cudaStream_t s);
struct LoraParams {
  const __nv_bfloat16* x;  // [M, ldx]
  long long ldx;
  const __nv_bfloat16* a;  // [slots, R, K]
  const __nv_bfloat16* b;  // [slots, N, R]
  const int* rank;         // [slots]
  const float* scale;      // [slots]
  const __nv_bfloat16* y;  // [M, ldy]
  long long ldy;
  __nv_bfloat16* out;      // [M, ldo]
  long long ldo;
  const int* order;
  const int4* tiles;
  const int* num_tiles;
  int M, K, N, R, tm, max_tiles;
  bool silu, in_place;
  __nv_bfloat16* h;  // [M, 2, R] scratch (tiles of 128 rows): scale * A x of every position, upper and lower part
  int* status;
};
cudaError_t lora_add_launch(const LoraParams& p, int num_sms, cudaStream_t s);

}  // namespace sq
