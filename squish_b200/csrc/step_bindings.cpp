// step_bindings.cpp — Python bindings of the serving-step operators (step_ops.h). Arguments are
// checked for device, dtype, shape and layout before the first CUDA call; every call launches on
// the current stream of its tensors' device and allocates nothing but lora_add's h (above 512 rows).
#include <torch/extension.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>

#include <string>

#include "step_ops.h"

namespace {

using OptTensor = c10::optional<torch::Tensor>;

// Numbers enter messages as strings: streaming an integer needs a locale facet, which a compiler whose
// libstdc++ differs from the interpreter's looks up in the wrong table (the message would crash).
std::string str(int64_t v) { return std::to_string(v); }

void check(const torch::Tensor& t, const char* name, torch::ScalarType dt, const torch::Device& dev) {
  TORCH_CHECK(t.is_cuda(), name, " must be a CUDA tensor");
  TORCH_CHECK(t.device() == dev, name, " is on ", t.device().str(), ", not on ", dev.str());
  TORCH_CHECK(t.scalar_type() == dt, name, " must be ", toString(dt), ", not ", toString(t.scalar_type()));
}
// a contiguous array of at least n elements
template <typename T>
T* arr(const torch::Tensor& t, const char* name, torch::ScalarType dt, const torch::Device& dev, int64_t n) {
  check(t, name, dt, dev);
  TORCH_CHECK(t.is_contiguous(), name, " must be contiguous");
  TORCH_CHECK(t.numel() >= n, name, " needs ", str(n), " elements, has ", str(t.numel()));
  return reinterpret_cast<T*>(t.data_ptr());
}
template <typename T>
T* opt_arr(const OptTensor& t, const char* name, torch::ScalarType dt, const torch::Device& dev, int64_t n) {
  return t.has_value() && t->defined() ? arr<T>(*t, name, dt, dev, n) : nullptr;
}
const torch::Device cuda_device(const torch::Tensor& t, const char* name) {
  TORCH_CHECK(t.is_cuda(), name, " must be a CUDA tensor");
  return t.device();
}
void ok(cudaError_t e, const char* what) {
  TORCH_CHECK(e == cudaSuccess, what, ": squish_b200 kernel launch failed: ", cudaGetErrorString(e));
}
cudaStream_t stream() { return at::cuda::getCurrentCUDAStream().stream(); }
int sms() { return at::cuda::getCurrentDeviceProperties()->multiProcessorCount; }

constexpr auto I32 = torch::kInt32;
constexpr auto F32 = torch::kFloat32;
constexpr auto BF16 = torch::kBFloat16;

// ------------------------------------------------------------------ step layout
void step_layout(torch::Tensor ctx, torch::Tensor q, torch::Tensor tables, torch::Tensor free_pages, int64_t page,
                 int64_t tile, torch::Tensor out, int64_t max_seqs, int64_t cap, int64_t tcap, torch::Tensor status) {
  const auto dev = cuda_device(ctx, "ctx_len");
  const int64_t B = ctx.numel();
  TORCH_CHECK(B >= 1 && B <= sq::kLayoutMaxSeqs, "a step has 1..", str(sq::kLayoutMaxSeqs), " sequences, not ", str(B));
  TORCH_CHECK(q.numel() == B, "q_len has ", str(q.numel()), " sequences, ctx_len ", str(B));
  TORCH_CHECK(page >= 1 && page <= (1 << 20), "page_size must be in 1..2^20");
  TORCH_CHECK(tile >= 1 && tile <= (1 << 20), "tile must be in 1..2^20");
  check(tables, "block_tables", I32, dev);
  TORCH_CHECK(tables.dim() == 2 && tables.size(0) == B && (tables.size(1) <= 1 || tables.stride(1) == 1) &&
                  (B == 1 || tables.stride(0) >= tables.size(1)) && tables.stride(0) <= INT32_MAX,
              "block_tables must be [sequences, pages] with unit page stride and rows of their own");
  sq::StepLayoutParams p{};
  p.ctx_len = arr<int>(ctx, "ctx_len", I32, dev, B);
  p.q_len = arr<int>(q, "q_len", I32, dev, B);
  p.block_tables = reinterpret_cast<int*>(tables.data_ptr());
  p.bt_stride = (int)tables.stride(0);
  p.bt_width = (int)tables.size(1);
  p.free_pages = arr<int>(free_pages, "free_pages", I32, dev, 0);
  TORCH_CHECK(cap >= 0 && tcap >= 0 && cap <= (1 << 28) && tcap <= (1 << 28) && free_pages.numel() <= (1 << 30),
              "step buffers above 2^28 rows");
  TORCH_CHECK(B <= max_seqs, "a step of ", str(B), " sequences in a layout of ", str(max_seqs));
  p.n_free = (int)free_pages.numel();
  p.B = (int)B;
  p.page_size = (int)page;
  p.tile = (int)tile;
  p.token_cap = (int)cap;
  p.tile_cap = (int)tcap;
  // (blocks read the lengths and the free list while others already write the results and the tables)
  auto share = [](const torch::Tensor& t, int64_t n, const torch::Tensor& u, int64_t m) {
    const uintptr_t a = reinterpret_cast<uintptr_t>(t.data_ptr()), b = reinterpret_cast<uintptr_t>(u.data_ptr());
    return n > 0 && m > 0 && a < b + 4 * m && b < a + 4 * n;
  };
  const int64_t table_n = tables.size(1) > 0 ? (B - 1) * tables.stride(0) + tables.size(1) : 0;
  auto apart = [&](const torch::Tensor& t, const char* name, int64_t n) {
    TORCH_CHECK(!share(t, n, out, out.numel()), name, " is part of the step layout it makes");
    TORCH_CHECK(!share(t, n, tables, table_n), name, " is part of block_tables");
  };
  apart(ctx, "ctx_len", B);
  apart(q, "q_len", B);
  apart(free_pages, "free_pages", free_pages.numel());
  TORCH_CHECK(!share(tables, table_n, out, out.numel()), "block_tables is part of the step layout it makes");
  // one buffer, its rows in this order, each padded to a multiple of four (ops.step.StepLayout)
  auto pad = [](int64_t n) { return (n + 3) / 4 * 4; };
  int* at = arr<int>(out, "the step layout", I32, dev,
                     pad(max_seqs + 1) + 2 * pad(max_seqs) + 4 + 3 * pad(cap) + 2 * pad(tcap));
  TORCH_CHECK(reinterpret_cast<uintptr_t>(at) % 16 == 0, "the step layout must be 16-byte aligned");
  auto row = [&](int64_t n) {
    int* r = at;
    at += pad(n);
    return r;
  };
  p.q_start = row(max_seqs + 1);
  p.kv_len = row(max_seqs);
  p.last_row = row(max_seqs);
  p.totals = row(3);
  p.positions = row(cap);
  p.slots = row(cap);
  p.token_seq = row(cap);
  p.tile_seq = row(tcap);
  p.tile_q0 = row(tcap);
  p.status = arr<int>(status, "status", I32, dev, 1);
  const c10::cuda::CUDAGuard g(dev);
  ok(sq::step_layout_launch(p, sms(), stream()), "step_layout");
}

// ------------------------------------------------------------------ scored routing
void moe_route_scored(torch::Tensor logits, int64_t K, torch::Tensor ids, torch::Tensor w, bool sigmoid, OptTensor bias,
                      int64_t groups, int64_t top_groups, bool top2, bool renorm, double scale) {
  const auto dev = cuda_device(logits, "logits");
  const bool f32 = logits.scalar_type() == F32;
  TORCH_CHECK(f32 || logits.scalar_type() == BF16, "logits must be bf16 or float32");
  TORCH_CHECK(logits.dim() == 2 && (logits.size(1) <= 1 || logits.stride(1) == 1),
              "logits must be [tokens, experts] with unit column stride");
  const int64_t T = logits.size(0), E = logits.size(1);
  TORCH_CHECK(E >= 1 && E <= sq::kRouteMaxExperts, "1..", str(sq::kRouteMaxExperts), " experts, not ", str(E));
  TORCH_CHECK(groups >= 1 && groups <= sq::kRouteMaxGroups && E % groups == 0, str(E), " experts do not split into ",
              str(groups), " groups (at most ", str(sq::kRouteMaxGroups), ")");
  TORCH_CHECK(top_groups >= 1 && top_groups <= groups, "top_groups must be in 1..", str(groups));
  TORCH_CHECK(K >= 1 && K <= sq::kRouteMaxK && K <= E / groups * top_groups, "top_k must be in 1..",
              str(std::min<int64_t>(sq::kRouteMaxK, E / groups * top_groups)), ", not ", str(K));
  TORCH_CHECK(T <= INT32_MAX / 64 && logits.stride(0) >= 0 && logits.stride(0) <= INT32_MAX, "too many tokens");
  sq::RouteScoredParams p{};
  p.logits = logits.data_ptr();
  p.ld = (int)logits.stride(0);
  p.T = (int)T;
  p.E = (int)E;
  p.K = (int)K;
  p.f32 = f32;
  p.sigmoid = sigmoid;
  p.bias = opt_arr<float>(bias, "bias", F32, dev, E);
  p.groups = (int)groups;
  p.top_groups = (int)top_groups;
  p.top2 = top2;
  p.renorm = renorm;
  p.scale = (float)scale;
  p.ids = arr<int>(ids, "ids", I32, dev, T * K);
  p.w = arr<float>(w, "weights", F32, dev, T * K);
  if (T == 0) return;
  const c10::cuda::CUDAGuard g(dev);
  ok(sq::moe_route_scored_launch(p, stream()), "moe_route_scored");
}

// ------------------------------------------------------------------ sampling
void sample_uniform(torch::Tensor logits, torch::Tensor uniforms, torch::Tensor out_tokens, OptTensor temperature,
                    OptTensor top_p, OptTensor top_k, OptTensor min_p, OptTensor allow_mask, OptTensor out_logprob) {
  const auto dev = cuda_device(logits, "logits");
  check(logits, "logits", BF16, dev);
  TORCH_CHECK(logits.dim() == 2 && (logits.size(1) <= 1 || logits.stride(1) == 1),
              "logits must be [rows, vocab] with unit column stride");
  const int64_t B = logits.size(0), V = logits.size(1);
  TORCH_CHECK(V >= 1 && V <= (1 << 26), "vocab must be in 1..2^26");
  TORCH_CHECK(B <= INT32_MAX && logits.stride(0) >= 0, "bad logits rows");
  const int64_t words = (V + 31) / 32;
  if (allow_mask.has_value() && allow_mask->defined())
    TORCH_CHECK(allow_mask->dim() == 2 && allow_mask->size(0) >= B && allow_mask->size(1) == words,
                "allow_mask must be [rows, ", str(words), "]");
  sq::SampleUniformParams p{};
  p.logits = reinterpret_cast<const __nv_bfloat16*>(logits.data_ptr());
  p.ld = logits.stride(0);
  p.V = (int)V;
  p.B = (int)B;
  p.uniforms = arr<float>(uniforms, "uniforms", F32, dev, B);
  p.temperature = opt_arr<float>(temperature, "temperature", F32, dev, B);
  p.top_p = opt_arr<float>(top_p, "top_p", F32, dev, B);
  p.top_k = opt_arr<int>(top_k, "top_k", I32, dev, B);
  p.min_p = opt_arr<float>(min_p, "min_p", F32, dev, B);
  p.allow_mask = opt_arr<uint32_t>(allow_mask, "allow_mask", I32, dev, B * words);
  p.out_tokens = arr<int>(out_tokens, "out_tokens", I32, dev, B);
  p.out_logprob = opt_arr<float>(out_logprob, "out_logprob", F32, dev, B);
  if (B == 0) return;
  const c10::cuda::CUDAGuard g(dev);
  ok(sq::sample_uniform_launch(p, sms(), stream()), "sample_uniform");
}

// ------------------------------------------------------------------ adapters
void lora_plan(torch::Tensor row_slot, int64_t slots, int64_t tm, torch::Tensor order, torch::Tensor tiles,
               torch::Tensor num_tiles, torch::Tensor status) {
  const auto dev = cuda_device(row_slot, "row_slots");
  const int64_t M = row_slot.numel();
  TORCH_CHECK(slots >= 1 && slots <= sq::kLoraMaxSlots, "1..", str(sq::kLoraMaxSlots), " adapter slots, not ", str(slots));
  TORCH_CHECK(tm == 16 || tm == 128, "tile rows must be 16 or 128");
  TORCH_CHECK(M <= (1 << 22), "at most 2^22 rows, not ", str(M));
  sq::LoraPlanParams p{};
  p.row_slot = arr<int>(row_slot, "row_slots", I32, dev, 0);
  p.M = (int)M;
  p.slots = (int)slots;
  p.tm = (int)tm;
  p.order = arr<int>(order, "order", I32, dev, M);
  p.max_tiles = (int)((M + tm - 1) / tm + std::min<int64_t>(slots + 1, M));
  p.tiles = arr<int4>(tiles, "tiles", I32, dev, (int64_t)p.max_tiles * 4);
  TORCH_CHECK(reinterpret_cast<uintptr_t>(p.tiles) % 16 == 0, "tiles must be 16-byte aligned");
  p.num_tiles = arr<int>(num_tiles, "num_tiles", I32, dev, 1);
  p.status = arr<int>(status, "status", I32, dev, 1);
  const c10::cuda::CUDAGuard g(dev);
  ok(sq::lora_plan_launch(p, stream()), "lora_plan");
}

const __nv_bfloat16* rows16(const torch::Tensor& t, const char* name, const torch::Device& dev, int64_t rows,
                            int64_t cols) {
  check(t, name, BF16, dev);
  TORCH_CHECK(t.dim() == 2 && t.size(0) == rows && t.size(1) == cols, name, " must be [", str(rows), ", ", str(cols), "]");
  TORCH_CHECK(t.stride(1) == 1 && t.stride(0) % 8 == 0 && t.stride(0) >= 0 &&
                  reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0,
              name, " rows must have unit column stride and be 16-byte aligned");
  return reinterpret_cast<const __nv_bfloat16*>(t.data_ptr());
}
// Do two bf16 matrices share memory? Column ranges of one buffer (rows of the same stride) do not.
bool overlap(const torch::Tensor& a, const torch::Tensor& b) {
  if (a.numel() == 0 || b.numel() == 0) return false;
  auto end = [](const torch::Tensor& t) {
    return reinterpret_cast<uintptr_t>(t.data_ptr()) + 2 * ((t.size(0) - 1) * t.stride(0) + t.size(1));
  };
  if (reinterpret_cast<uintptr_t>(a.data_ptr()) >= end(b) || reinterpret_cast<uintptr_t>(b.data_ptr()) >= end(a))
    return false;
  const int64_t ld = a.stride(0);
  if (ld != b.stride(0) || ld <= 0 || a.size(0) <= 1 || b.size(0) <= 1) return true;
  const int64_t d = (reinterpret_cast<intptr_t>(a.data_ptr()) - reinterpret_cast<intptr_t>(b.data_ptr())) / 2;
  const int64_t col = ((d % ld) + ld) % ld;  // first column of a in rows that start at b's
  return col < b.size(1) || col + a.size(1) > ld;
}

void lora_add(torch::Tensor x, torch::Tensor a, torch::Tensor b, torch::Tensor rank, torch::Tensor scale,
              torch::Tensor y, torch::Tensor out, torch::Tensor order, torch::Tensor tiles, torch::Tensor num_tiles,
              int64_t tm, int64_t slots, int64_t max_tiles, bool silu, torch::Tensor status) {
  const auto dev = cuda_device(x, "x");
  check(a, "pool a", BF16, dev);
  check(b, "pool b", BF16, dev);
  TORCH_CHECK(a.dim() == 3 && b.dim() == 3 && a.size(0) == b.size(0) && a.size(1) == b.size(2) && a.is_contiguous() &&
                  b.is_contiguous(),
              "the pool holds a [slots, rank, k] and b [slots, n, rank]");
  TORCH_CHECK(a.size(0) == slots, "the plan is for ", str(slots), " adapter slots, the pool has ", str(a.size(0)));
  const int64_t M = order.numel(), K = a.size(2), N = b.size(1), R = a.size(1);
  TORCH_CHECK(R == 16 || R == 32 || R == 64 || R == 128, "pool rank must be 16, 32, 64 or 128");
  TORCH_CHECK(K % 8 == 0 && K >= 8 && N % 8 == 0 && N >= 8, "k and n must be multiples of 8");
  TORCH_CHECK(!silu || N % 128 == 0, "the SiLU*up epilogue needs [gate 64 | up 64] blocks: n a multiple of 128");
  sq::LoraParams p{};
  p.x = rows16(x, "x", dev, M, K);
  p.y = rows16(y, "y", dev, M, N);
  p.out = const_cast<__nv_bfloat16*>(rows16(out, "out", dev, M, silu ? N / 2 : N));
  TORCH_CHECK(M <= 1 || out.stride(0) >= out.size(1), "out rows overlap");
  p.in_place = !silu && out.data_ptr() == y.data_ptr() && (M <= 1 || out.stride(0) == y.stride(0));
  TORCH_CHECK(p.in_place || !overlap(out, y), "out overlaps y (the same tensor is allowed, without the epilogue)");
  TORCH_CHECK(!overlap(out, x), "out overlaps x");
  p.ldx = x.stride(0);
  p.ldy = y.stride(0);
  p.ldo = out.stride(0);
  p.a = reinterpret_cast<const __nv_bfloat16*>(a.data_ptr());
  p.b = reinterpret_cast<const __nv_bfloat16*>(b.data_ptr());
  p.rank = arr<int>(rank, "rank", I32, dev, slots);
  p.scale = arr<float>(scale, "scale", F32, dev, slots);
  p.order = arr<int>(order, "order", I32, dev, M);
  p.tiles = arr<int4>(tiles, "tiles", I32, dev, max_tiles * 4);
  p.num_tiles = arr<int>(num_tiles, "num_tiles", I32, dev, 1);
  p.M = (int)M;
  p.K = (int)K;
  p.N = (int)N;
  p.R = (int)R;
  p.tm = (int)tm;
  p.max_tiles = (int)max_tiles;
  p.silu = silu;
  p.status = arr<int>(status, "status", I32, dev, 1);
  if (M == 0) return;
  const c10::cuda::CUDAGuard g(dev);
  torch::Tensor h;  // from the caching allocator, in this stream's order: calls never share it
  if (tm != 16) {
    h = torch::empty({M, 2, R}, x.options());
    p.h = reinterpret_cast<__nv_bfloat16*>(h.data_ptr());
  }
  ok(sq::lora_add_launch(p, sms(), stream()), "lora_add");
}

}  // namespace

namespace sqstep {

void register_step(pybind11::module& m) {
  m.def("step_layout", &step_layout);
  m.def("moe_route_scored", &moe_route_scored);
  m.def("sample_uniform", &sample_uniform);
  m.def("lora_plan", &lora_plan);
  m.def("lora_add", &lora_add);
}

}  // namespace sqstep
