// bindings.cpp -- torch extension `decode_kernel._cuda`, a thin layer over the
// C ABI in include/dk_w4a16.h.
//
// Keeps the reference module's exports, argument names, defaults and error
// messages (RohanDisa/decode-kernel csrc/bindings.cpp:10-48, 114-129) so code
// and tests written against the reference run unchanged:
//   w4a16_gemv(packed, scales, x, version=5, split_k=4, reuse_weights=False,
//              warps_per_row=1) -> fp16 [B, M]
//   d2d_copy(src, dst), stream_read(src, partials), stream_write(dst),
//   stream_recommended_blocks(), last_kernel_stamp()
// and adds: w4a16_gemv_out (caller-provided y, optional PDL launch),
// workspace_bytes, quantize_pack / unpack_to_int / dequantize on the GPU,
// device_error, and the rest of a decode step: Cache8 (a paged 8-bit cache's
// tensors, checked once), cache_plan, cache_append, cache_attention, block_norm.
// Every C-ABI status other than DK_OK becomes a RuntimeError.
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGraphsC10Utils.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/extension.h>

#include <algorithm>
#include <array>
#include <cmath>
#include <cstdint>
#include <map>
#include <mutex>
#include <optional>
#include <string>
#include <tuple>
#include <utility>
#include <vector>

#include "dk_w4a16.h"

namespace {

void check_status(dk_status s, const char* what) {
  if (s == DK_OK) return;
  std::string msg = std::string(what) + ": " + dk_status_string(s);
  if (s == DK_ERR_LAUNCH || s == DK_ERR_CUDA) msg += std::string(" [") + dk_last_cuda_error() + "]";
  TORCH_CHECK(false, msg);
}

bool aligned16(const torch::Tensor& t) {
  return (reinterpret_cast<uintptr_t>(t.data_ptr()) & 15u) == 0;
}

// bindings.cpp:10-33
void check_gemv_inputs(const torch::Tensor& packed, const torch::Tensor& scales,
                       const torch::Tensor& x) {
  TORCH_CHECK(packed.is_cuda() && scales.is_cuda() && x.is_cuda(),
              "packed, scales, and x must be CUDA tensors");
  TORCH_CHECK(packed.scalar_type() == torch::kInt32, "packed must be int32 (uint32 bit pattern)");
  TORCH_CHECK(scales.scalar_type() == torch::kFloat16, "scales must be fp16");
  TORCH_CHECK(x.scalar_type() == torch::kFloat16, "x must be fp16");
  TORCH_CHECK(packed.dim() == 2 && scales.dim() == 2 && x.dim() == 2,
              "packed [M,K/8], scales [M,K/128], x [B,K]");
  TORCH_CHECK(packed.is_contiguous() && scales.is_contiguous() && x.is_contiguous(),
              "packed, scales, and x must be contiguous");
  const int64_t M = packed.size(0);
  const int64_t K = packed.size(1) * DK_NIBBLES_PER_WORD;
  TORCH_CHECK(K % DK_GROUP_SIZE == 0, "K must be divisible by group size 128");
  TORCH_CHECK(scales.size(0) == M && scales.size(1) == K / DK_GROUP_SIZE,
              "scales shape must be [M, K/128]");
  TORCH_CHECK(x.size(1) == K, "x.shape[1] must equal K");
  TORCH_CHECK(packed.device() == scales.device() && packed.device() == x.device(),
              "packed, scales, and x must be on the same device");
  TORCH_CHECK(M <= INT32_MAX && K <= INT32_MAX && x.size(0) <= INT32_MAX,
              "dimensions must fit in int32");
}

// bindings.cpp:41-48
dk_gemv_config make_config(int version, int split_k, bool reuse_weights, int warps_per_row,
                           bool pdl) {
  TORCH_CHECK(version >= 0 && version <= 5, "version must be 0..5");
  TORCH_CHECK(split_k >= 1 && split_k <= 32, "split_k must be in [1, 32]");
  TORCH_CHECK(warps_per_row >= 1 && warps_per_row <= 8, "warps_per_row must be in [1, 8]");
  if (warps_per_row > 1) {
    TORCH_CHECK(version == 1 && !reuse_weights,
                "warps_per_row > 1 is implemented for streaming v1 only");
  }
  dk_gemv_config cfg;
  dk_gemv_config_init(&cfg);
  cfg.version = version;
  cfg.split_k = split_k;
  cfg.reuse_weights = reuse_weights ? 1 : 0;
  cfg.warps_per_row = warps_per_row;
  cfg.flags = pdl ? DK_FLAG_PDL : 0u;
  return cfg;
}

void run_gemv(const torch::Tensor& packed_in, const torch::Tensor& scales,
              const torch::Tensor& x_in, torch::Tensor& y, const dk_gemv_config& cfg) {
  // The kernels stream with 128-bit loads: re-home a (rare) misaligned view.
  const torch::Tensor packed = aligned16(packed_in) ? packed_in : packed_in.clone();
  const torch::Tensor x = aligned16(x_in) ? x_in : x_in.clone();
  const int M = static_cast<int>(packed.size(0));
  const int K = static_cast<int>(packed.size(1) * DK_NIBBLES_PER_WORD);
  const int B = static_cast<int>(x.size(0));
  const size_t ws_bytes = dk_w4a16_workspace_bytes(M, K, B, &cfg);
  torch::Tensor ws;
  if (ws_bytes) ws = torch::empty({static_cast<int64_t>(ws_bytes)}, x.options().dtype(torch::kUInt8));
  check_status(
      dk_w4a16_gemv(packed.data_ptr<int32_t>(),
                    reinterpret_cast<const uint16_t*>(scales.data_ptr<at::Half>()),
                    reinterpret_cast<const uint16_t*>(x.data_ptr<at::Half>()),
                    reinterpret_cast<uint16_t*>(y.data_ptr<at::Half>()), M, K, B, &cfg,
                    ws_bytes ? ws.data_ptr() : nullptr, ws_bytes,
                    at::cuda::getCurrentCUDAStream().stream()),
      "w4a16_gemv");
}

torch::Tensor w4a16_gemv(torch::Tensor packed, torch::Tensor scales, torch::Tensor x,
                         int version, int split_k, bool reuse_weights, int warps_per_row) {
  check_gemv_inputs(packed, scales, x);
  const dk_gemv_config cfg = make_config(version, split_k, reuse_weights, warps_per_row, false);
  const c10::cuda::CUDAGuard guard(x.device());
  auto y = torch::empty({x.size(0), packed.size(0)}, x.options());
  run_gemv(packed, scales, x, y, cfg);
  return y;
}

void w4a16_gemv_out(torch::Tensor packed, torch::Tensor scales, torch::Tensor x, torch::Tensor y,
                    int version, int split_k, bool reuse_weights, int warps_per_row, bool pdl) {
  check_gemv_inputs(packed, scales, x);
  TORCH_CHECK(y.is_cuda() && y.device() == x.device(), "y must be on x's device");
  TORCH_CHECK(y.scalar_type() == torch::kFloat16 && y.is_contiguous(), "y must be contiguous fp16");
  TORCH_CHECK(y.dim() == 2 && y.size(0) == x.size(0) && y.size(1) == packed.size(0),
              "y must be [B, M]");
  const dk_gemv_config cfg = make_config(version, split_k, reuse_weights, warps_per_row, pdl);
  const c10::cuda::CUDAGuard guard(x.device());
  run_gemv(packed, scales, x, y, cfg);
}

int64_t workspace_bytes(int64_t M, int64_t K, int64_t B, int version, int split_k,
                        bool reuse_weights) {
  const dk_gemv_config cfg = make_config(version, split_k, reuse_weights, 1, false);
  return static_cast<int64_t>(dk_w4a16_workspace_bytes(static_cast<int>(M), static_cast<int>(K),
                                                       static_cast<int>(B), &cfg));
}

// bindings.cpp:80-110
void d2d_copy(torch::Tensor src, torch::Tensor dst) {
  TORCH_CHECK(src.is_cuda() && dst.is_cuda(), "src and dst must be CUDA");
  TORCH_CHECK(src.nbytes() == dst.nbytes(), "src/dst size mismatch");
  TORCH_CHECK(src.nbytes() % 16 == 0, "copy size must be a multiple of 16");
  const c10::cuda::CUDAGuard guard(src.device());
  check_status(dk_d2d_copy(src.data_ptr(), dst.data_ptr(), src.nbytes(),
                           at::cuda::getCurrentCUDAStream().stream()),
               "d2d_copy");
}

void stream_read(torch::Tensor src, torch::Tensor partials) {
  TORCH_CHECK(src.is_cuda() && partials.is_cuda(), "src and partials must be CUDA");
  TORCH_CHECK(src.nbytes() % 16 == 0, "buffer size must be a multiple of 16");
  TORCH_CHECK(partials.scalar_type() == torch::kFloat32, "partials must be fp32");
  TORCH_CHECK(partials.is_contiguous(), "partials must be contiguous");
  const int blocks = static_cast<int>(partials.numel());
  TORCH_CHECK(blocks >= 1, "partials must have one float per block");
  const c10::cuda::CUDAGuard guard(src.device());
  check_status(dk_stream_read(src.data_ptr(), partials.data_ptr<float>(), src.nbytes(), blocks,
                              at::cuda::getCurrentCUDAStream().stream()),
               "stream_read");
}

void stream_write(torch::Tensor dst) {
  TORCH_CHECK(dst.is_cuda(), "dst must be CUDA");
  TORCH_CHECK(dst.nbytes() % 16 == 0, "buffer size must be a multiple of 16");
  const c10::cuda::CUDAGuard guard(dst.device());
  check_status(dk_stream_write(dst.data_ptr(), dst.nbytes(), dk_stream_recommended_blocks(-1),
                               at::cuda::getCurrentCUDAStream().stream()),
               "stream_write");
}

int stream_recommended_blocks() { return dk_stream_recommended_blocks(-1); }

int last_kernel_stamp() { return dk_last_kernel_stamp(-1); }

int device_error(bool clear) { return dk_device_error(-1, clear ? 1 : 0); }

std::vector<torch::Tensor> quantize_pack(torch::Tensor w, bool torch_cuda_scale) {
  TORCH_CHECK(w.is_cuda() && w.scalar_type() == torch::kFloat32 && w.dim() == 2,
              "weight must be a 2-D fp32 CUDA tensor");
  const int64_t M = w.size(0), K = w.size(1);
  TORCH_CHECK(K % DK_GROUP_SIZE == 0, "K=", K, " is not divisible by group_size=", DK_GROUP_SIZE);
  TORCH_CHECK(M <= INT32_MAX && K <= INT32_MAX, "dimensions must fit in int32");
  const c10::cuda::CUDAGuard guard(w.device());
  torch::Tensor wc = w.contiguous();
  if (!aligned16(wc)) wc = wc.clone();
  auto packed = torch::empty({M, K / DK_NIBBLES_PER_WORD}, w.options().dtype(torch::kInt32));
  auto scales = torch::empty({M, K / DK_GROUP_SIZE}, w.options().dtype(torch::kFloat16));
  check_status(dk_quantize_pack(wc.data_ptr<float>(), static_cast<int>(M), static_cast<int>(K),
                                packed.data_ptr<int32_t>(),
                                reinterpret_cast<uint16_t*>(scales.data_ptr<at::Half>()),
                                torch_cuda_scale ? DK_QUANT_TORCH_CUDA_SCALE : 0u,
                                at::cuda::getCurrentCUDAStream().stream()),
               "quantize_pack");
  return {packed, scales};
}

torch::Tensor unpack_to_int(torch::Tensor packed) {
  TORCH_CHECK(packed.is_cuda() && packed.scalar_type() == torch::kInt32 && packed.dim() == 2,
              "packed must be a 2-D int32 CUDA tensor");
  const int64_t M = packed.size(0), K = packed.size(1) * DK_NIBBLES_PER_WORD;
  TORCH_CHECK(K % DK_GROUP_SIZE == 0, "K must be divisible by group size 128");
  const c10::cuda::CUDAGuard guard(packed.device());
  auto pc = packed.contiguous();
  auto q = torch::empty({M, K}, packed.options());
  check_status(dk_unpack_to_int(pc.data_ptr<int32_t>(), static_cast<int>(M), static_cast<int>(K),
                                q.data_ptr<int32_t>(), at::cuda::getCurrentCUDAStream().stream()),
               "unpack_to_int");
  return q;
}

torch::Tensor dequantize(torch::Tensor packed, torch::Tensor scales) {
  TORCH_CHECK(packed.is_cuda() && scales.is_cuda(), "packed and scales must be CUDA tensors");
  TORCH_CHECK(packed.scalar_type() == torch::kInt32 && scales.scalar_type() == torch::kFloat16,
              "packed int32, scales fp16");
  const int64_t M = packed.size(0), K = packed.size(1) * DK_NIBBLES_PER_WORD;
  TORCH_CHECK(K % DK_GROUP_SIZE == 0 && scales.size(0) == M && scales.size(1) == K / DK_GROUP_SIZE,
              "scales shape must be [M, K/128]");
  const c10::cuda::CUDAGuard guard(packed.device());
  auto pc = packed.contiguous();
  auto sc = scales.contiguous();
  auto w = torch::empty({M, K}, packed.options().dtype(torch::kFloat32));
  check_status(dk_dequantize(pc.data_ptr<int32_t>(),
                             reinterpret_cast<const uint16_t*>(sc.data_ptr<at::Half>()),
                             static_cast<int>(M), static_cast<int>(K), w.data_ptr<float>(),
                             at::cuda::getCurrentCUDAStream().stream()),
               "dequantize");
  return w;
}

// ---------------------------------------------------------------------------
// The paged 8-bit cache and the norms between blocks.
// ---------------------------------------------------------------------------
using OptTensor = std::optional<torch::Tensor>;

// A cache's four tensors and their description, checked once.
struct Cache8 {
  torch::Tensor k, v, k_scale, v_scale;
  dk_cache8 c;

  Cache8(torch::Tensor k_, torch::Tensor v_, torch::Tensor ks, torch::Tensor vs)
      : k(std::move(k_)), v(std::move(v_)), k_scale(std::move(ks)), v_scale(std::move(vs)) {
    TORCH_CHECK(k.is_cuda() && v.is_cuda() && k_scale.is_cuda() && v_scale.is_cuda(),
                "the cache's tensors must be CUDA tensors");
    TORCH_CHECK(k.device() == v.device() && k.device() == k_scale.device() &&
                    k.device() == v_scale.device(),
                "the cache's tensors must be on one device");
    TORCH_CHECK(k.scalar_type() == v.scalar_type() &&
                    (k.scalar_type() == torch::kInt8 || k.scalar_type() == torch::kFloat8_e4m3fn),
                "k and v must both be int8 or both float8_e4m3fn");
    TORCH_CHECK(k.dim() == 4 && v.sizes() == k.sizes(),
                "k and v must be [blocks, kv_heads, block_size, head_dim]");
    TORCH_CHECK(k.size(0) >= 1 && k.size(0) <= INT32_MAX && k.size(1) >= 1 && k.size(1) <= 65535,
                "blocks and kv_heads out of range");
    TORCH_CHECK(k.size(2) >= 16 && k.size(2) <= 256 && k.size(2) % 16 == 0,
                "block_size must be a multiple of 16 in 16..256");
    TORCH_CHECK(k.size(3) == 64 || k.size(3) == 128 || k.size(3) == 256,
                "head_dim must be 64, 128 or 256");
    TORCH_CHECK(k.stride(3) == 1 && v.stride(3) == 1, "head_dim must be contiguous");
    for (int i = 0; i < 3; ++i)
      TORCH_CHECK(k.stride(i) % 32 == 0 && v.stride(i) % 32 == 0 && k.stride(i) >= 0 &&
                      v.stride(i) >= 0,
                  "the cache's strides must be multiples of 32");
    TORCH_CHECK((reinterpret_cast<uintptr_t>(k.data_ptr()) & 31u) == 0 &&
                    (reinterpret_cast<uintptr_t>(v.data_ptr()) & 31u) == 0,
                "k and v must be 32-byte aligned");
    TORCH_CHECK(k_scale.scalar_type() == torch::kFloat32 && v_scale.scalar_type() == torch::kFloat32,
                "scales must be fp32");
    for (const torch::Tensor* s : {&k_scale, &v_scale})
      TORCH_CHECK(s->dim() == 2 && s->size(0) == k.size(0) && s->size(1) == k.size(1) &&
                      s->is_contiguous(),
                  "scales must be contiguous [blocks, kv_heads]");
    c.k = k.data_ptr();
    c.v = v.data_ptr();
    c.k_scale = k_scale.data_ptr<float>();
    c.v_scale = v_scale.data_ptr<float>();
    c.blocks = static_cast<int>(k.size(0));
    c.kv_heads = static_cast<int>(k.size(1));
    c.block_size = static_cast<int>(k.size(2));
    c.head_dim = static_cast<int>(k.size(3));
    c.code = k.scalar_type() == torch::kInt8 ? DK_INT8 : DK_E4M3;
    c.k_block_stride = k.stride(0);
    c.k_head_stride = k.stride(1);
    c.k_token_stride = k.stride(2);
    c.v_block_stride = v.stride(0);
    c.v_head_stride = v.stride(1);
    c.v_token_stride = v.stride(2);
  }
};

dk_dtype half_type(const torch::Tensor& t, const char* what) {
  if (t.scalar_type() == torch::kFloat16) return DK_FP16;
  TORCH_CHECK(t.scalar_type() == torch::kBFloat16, what, " must be fp16 or bf16");
  return DK_BF16;
}

void check_ints(const torch::Tensor& t, torch::ScalarType type, int64_t n, const torch::Device& device,
                const char* what) {
  TORCH_CHECK(t.is_cuda() && t.device() == device, what, " must be on the call's CUDA device");
  TORCH_CHECK(t.scalar_type() == type, what, " must be ", type);
  TORCH_CHECK(t.dim() == 1 && t.size(0) == n && t.is_contiguous(), what, " must be contiguous [" + std::to_string(n) + "]");
}

void check_table(const torch::Tensor& t, int64_t requests, const torch::Device& device) {
  TORCH_CHECK(t.is_cuda() && t.device() == device, "block_table must be on the call's CUDA device");
  TORCH_CHECK(t.scalar_type() == torch::kInt32 && t.dim() == 2 && t.size(0) == requests &&
                  t.size(1) >= 1 && t.stride(1) == 1 && t.stride(0) >= t.size(1) &&
                  t.stride(0) <= INT32_MAX,
              "block_table must be int32 [requests, max_blocks] with contiguous rows");
}

// A tensor over part of another's storage, without the dispatcher's work of a
// view (a plan makes four small tensors every step).
torch::Tensor part_of(const torch::Tensor& whole, torch::ScalarType type, int64_t byte, c10::IntArrayRef sizes) {
  torch::Tensor t = at::detail::make_tensor<c10::TensorImpl>(
      c10::Storage(whole.storage()), whole.key_set(), c10::scalarTypeToTypeMeta(type));
  t.unsafeGetTensorImpl()->set_storage_offset(byte / static_cast<int64_t>(c10::elementSize(type)));
  t.unsafeGetTensorImpl()->set_sizes_contiguous(sizes);
  return t;
}

std::tuple<torch::Tensor, torch::Tensor, torch::Tensor, torch::Tensor> cache_plan(
    torch::Tensor held, torch::Tensor fresh, torch::Tensor block_table, torch::Tensor free_blocks,
    torch::Tensor ring, int64_t block_size, int64_t tokens, OptTensor lengths, OptTensor starts,
    OptTensor slots, OptTensor ring_out) {
  TORCH_CHECK(held.is_cuda(), "held must be a CUDA tensor");
  TORCH_CHECK(held.dim() == 1, "held must be [requests]");
  const torch::Device device = held.device();
  const int64_t n = held.size(0);
  TORCH_CHECK(n <= DK_PLAN_MAX_REQUESTS, "at most " + std::to_string(DK_PLAN_MAX_REQUESTS) + " requests");
  TORCH_CHECK(tokens >= 0 && tokens <= INT32_MAX, "tokens out of range");
  TORCH_CHECK(block_size >= 16 && block_size <= 256 && block_size % 16 == 0,
              "block_size must be a multiple of 16 in 16..256");
  check_ints(held, torch::kInt32, n, device, "held");
  check_ints(fresh, torch::kInt32, n, device, "fresh");
  check_table(block_table, n, device);
  TORCH_CHECK(free_blocks.numel() <= INT32_MAX, "free_blocks is too long");
  check_ints(free_blocks, torch::kInt32, free_blocks.numel(), device, "free_blocks");
  check_ints(ring, torch::kInt64, 4, device, "ring");
  const c10::cuda::CUDAGuard guard(device);
  // What is not given lies in one allocation: slots, ring, lengths, starts.
  const int64_t ring_at = (8 * tokens + 15) / 16 * 16, lengths_at = ring_at + 32,
                starts_at = lengths_at + 4 * n, bytes = starts_at + 4 * (n + 1);
  torch::Tensor whole;
  if (!lengths || !starts || !slots || !ring_out)
    whole = torch::empty({bytes}, held.options().dtype(torch::kUInt8));
  auto given = [&](OptTensor& t, torch::ScalarType type, int64_t at, int64_t size, const char* what) {
    if (!t) return part_of(whole, type, at, {size});
    check_ints(*t, type, size, device, what);
    return *t;
  };
  torch::Tensor l = given(lengths, torch::kInt32, lengths_at, n, "lengths");
  torch::Tensor s = given(starts, torch::kInt32, starts_at, n + 1, "starts");
  torch::Tensor m = given(slots, torch::kInt64, 0, tokens, "slots");
  torch::Tensor r = given(ring_out, torch::kInt64, ring_at, 4, "ring_out");
  check_status(
      dk_cache_plan(held.data_ptr<int32_t>(), fresh.data_ptr<int32_t>(), static_cast<int>(n),
                    block_table.data_ptr<int32_t>(), static_cast<int>(block_table.size(1)),
                    static_cast<int>(n > 1 ? block_table.stride(0) : block_table.size(1)),
                    static_cast<int>(block_size), free_blocks.data_ptr<int32_t>(),
                    static_cast<int>(free_blocks.numel()), ring.data_ptr<int64_t>(),
                    r.data_ptr<int64_t>(), l.data_ptr<int32_t>(), s.data_ptr<int32_t>(),
                    m.data_ptr<int64_t>(), static_cast<int>(tokens),
                    at::cuda::getCurrentCUDAStream().stream()),
      "cache_plan");
  return {l, s, m, r};
}

void cache_append(torch::Tensor k, torch::Tensor v, torch::Tensor slots, const Cache8& cache) {
  const torch::Device device = cache.k.device();
  TORCH_CHECK(k.is_cuda() && v.is_cuda() && k.device() == device && v.device() == device,
              "k and v must be CUDA tensors on the cache's device");
  TORCH_CHECK(k.dim() == 3 && k.size(1) == cache.c.kv_heads && k.size(2) == cache.c.head_dim,
              "k must be [tokens, kv_heads, head_dim]");
  TORCH_CHECK(v.sizes() == k.sizes() && v.scalar_type() == k.scalar_type(),
              "v must have k's shape and type");
  TORCH_CHECK(k.size(0) <= INT32_MAX, "too many tokens");
  const dk_dtype type = half_type(k, "k and v");
  check_ints(slots, torch::kInt64, k.size(0), device, "slots");
  const c10::cuda::CUDAGuard guard(device);
  // The kernel reads 8 values at once: re-home views that do not allow it.
  auto fits = [&](const torch::Tensor& t) {
    return t.stride(2) == 1 && t.stride(0) % 8 == 0 && t.stride(1) % 8 == 0 && aligned16(t);
  };
  const torch::Tensor kc = fits(k) ? k : k.clone(at::MemoryFormat::Contiguous);
  const torch::Tensor vc = fits(v) ? v : v.clone(at::MemoryFormat::Contiguous);
  check_status(dk_cache_append(&cache.c, kc.data_ptr(), vc.data_ptr(), type,
                               static_cast<int>(k.size(0)), kc.stride(0), kc.stride(1),
                               vc.stride(0), vc.stride(1), slots.data_ptr<int64_t>(),
                               at::cuda::getCurrentCUDAStream().stream()),
               "cache_append");
}

// The attention workspaces: one for each device and stream, of the largest head
// size that the stream has asked for (the counters lie in the same place for all),
// its counters zeroed when it is made; every call leaves it ready for the next on
// that stream.  They stay until release_workspaces(): a dropped one goes back to
// the caching allocator, which gives it out again in its stream's order.  A call that is being captured gets one of its own with the counters'
// zeroing (a few KB of some 24 MB) in the graph, since the graph may be replayed
// beside later calls of the stream.
struct Workspaces {
  std::mutex mu;
  std::map<std::pair<int, cudaStream_t>, torch::Tensor> of;
};
Workspaces& workspaces() {
  static auto* w = new Workspaces();  // never destroyed: the process may end after the CUDA context
  return *w;
}

torch::Tensor attention_workspace(int head_dim, const at::cuda::CUDAStream& stream) {
  const int64_t bytes = static_cast<int64_t>(dk_cache_attention_workspace_bytes(head_dim));
  auto make = [&] {
    const torch::Tensor w = torch::empty({bytes}, torch::TensorOptions().dtype(torch::kUInt8).device(stream.device()));
    C10_CUDA_CHECK(cudaMemsetAsync(w.data_ptr(), 0, dk_cache_attention_counter_bytes(), stream.stream()));
    return w;
  };
  if (c10::cuda::currentStreamCaptureStatusMayInitCtx() != c10::cuda::CaptureStatus::None) return make();
  Workspaces& kept = workspaces();
  const std::lock_guard<std::mutex> lock(kept.mu);
  torch::Tensor& w = kept.of[{stream.device_index(), stream.stream()}];
  if (!w.defined() || w.numel() < bytes) w = make();
  return w;
}

void release_workspaces() {
  Workspaces& kept = workspaces();
  const std::lock_guard<std::mutex> lock(kept.mu);
  kept.of.clear();
}

std::tuple<torch::Tensor, OptTensor> cache_attention(torch::Tensor q, const Cache8& cache,
                                                     torch::Tensor block_table, torch::Tensor lengths,
                                                     OptTensor starts, std::optional<double> scale,
                                                     bool causal, int64_t window, OptTensor out,
                                                     bool want_lse) {
  const torch::Device device = cache.k.device();
  TORCH_CHECK(q.is_cuda() && q.device() == device, "q must be a CUDA tensor on the cache's device");
  TORCH_CHECK(q.dim() == 3 && q.size(2) == cache.c.head_dim, "q must be [tokens, q_heads, head_dim]");
  TORCH_CHECK(q.size(0) <= INT32_MAX && q.size(1) >= 1 && q.size(1) % cache.c.kv_heads == 0 &&
                  q.size(1) <= INT32_MAX,
              "q_heads must be a multiple of kv_heads");
  TORCH_CHECK(window >= 0 && window <= INT32_MAX && (window == 0 || causal),
              "window must be 0 (none) or positive, and causal");
  const int64_t n = lengths.size(0);
  TORCH_CHECK(n <= INT32_MAX, "too many requests");
  check_ints(lengths, torch::kInt32, n, device, "lengths");
  check_table(block_table, n, device);
  if (starts) check_ints(*starts, torch::kInt32, n + 1, device, "starts");
  else TORCH_CHECK(q.size(0) == n, "without starts q must have one token for each request");
  const c10::cuda::CUDAGuard guard(device);
  dk_cache_attention_args a;
  a.dtype = half_type(q, "q");
  const bool fits = q.stride(2) == 1 && q.stride(0) % 8 == 0 && q.stride(1) % 8 == 0 && aligned16(q);
  const torch::Tensor qc = fits ? q : q.clone(at::MemoryFormat::Contiguous);
  torch::Tensor o;
  if (out) {
    o = *out;
    TORCH_CHECK(o.is_cuda() && o.device() == device && o.scalar_type() == q.scalar_type() &&
                    o.sizes() == q.sizes() && o.is_contiguous() && aligned16(o),
                "out must be contiguous, with q's shape, type and device");
  } else {
    o = torch::empty(q.sizes(), q.options());
  }
  OptTensor lse;
  if (want_lse) lse = torch::empty({q.size(0), q.size(1)}, q.options().dtype(torch::kFloat32));
  const at::cuda::CUDAStream stream = at::cuda::getCurrentCUDAStream();
  const torch::Tensor ws = attention_workspace(cache.c.head_dim, stream);
  a.cache = cache.c;
  a.q = qc.data_ptr();
  a.out = o.data_ptr();
  a.lse = want_lse ? lse->data_ptr<float>() : nullptr;
  a.q_token_stride = qc.stride(0);
  a.q_head_stride = qc.stride(1);
  a.block_table = block_table.data_ptr<int32_t>();
  a.max_blocks = static_cast<int>(block_table.size(1));
  a.table_stride = static_cast<int>(n > 1 ? block_table.stride(0) : block_table.size(1));
  a.lengths = lengths.data_ptr<int32_t>();
  a.starts = starts ? starts->data_ptr<int32_t>() : nullptr;
  a.requests = static_cast<int>(n);
  a.tokens = static_cast<int>(q.size(0));
  a.q_heads = static_cast<int>(q.size(1));
  a.scale = static_cast<float>(scale ? *scale : 1.0 / std::sqrt(static_cast<double>(cache.c.head_dim)));
  a.causal = causal ? 1 : 0;
  a.window = static_cast<int>(window);
  check_status(dk_cache_attention(&a, ws.data_ptr(), static_cast<size_t>(ws.numel()), stream.stream()),
               "cache_attention");
  return {o, lse};
}

std::tuple<torch::Tensor, OptTensor> block_norm(torch::Tensor residual, OptTensor y, int kind,
                                                OptTensor post_weight, OptTensor post_bias,
                                                OptTensor gate, int act, double residual_scale,
                                                double block_scale, OptTensor pre_weight,
                                                OptTensor pre_bias, double eps, bool inplace) {
  TORCH_CHECK(residual.is_cuda(), "residual must be a CUDA tensor");
  TORCH_CHECK(residual.dim() >= 1 && residual.size(-1) >= 1 && residual.size(-1) <= 32768,
              "residual must be [..., dim] with dim in 1..32768");
  TORCH_CHECK(y || pre_weight, "nothing to do: neither y nor pre_weight");
  TORCH_CHECK(y || !(gate || post_weight), "gate and post_weight belong to y");
  TORCH_CHECK(post_weight || !post_bias, "post_bias needs post_weight");
  TORCH_CHECK(pre_weight || !pre_bias, "pre_bias needs pre_weight");
  const torch::Device device = residual.device();
  const int64_t dim = residual.size(-1), rows = residual.numel() / dim;
  TORCH_CHECK(rows <= INT32_MAX, "too many rows");
  dk_block_norm_args a{};
  a.dtype = half_type(y ? *y : *pre_weight, "y and the weights");
  const torch::ScalarType type = y ? y->scalar_type() : pre_weight->scalar_type();
  TORCH_CHECK(residual.scalar_type() == type || residual.scalar_type() == torch::kFloat32,
              "residual must have y's type or be fp32");
  a.residual_dtype = residual.scalar_type() == torch::kFloat32 ? DK_FP32 : a.dtype;
  auto weight = [&](const OptTensor& t, const char* what) -> const void* {
    if (!t) return nullptr;
    TORCH_CHECK(t->is_cuda() && t->device() == device && t->scalar_type() == type && t->dim() == 1 &&
                    t->size(0) == dim && t->is_contiguous(),
                what, " must be contiguous [dim] with y's type, on residual's device");
    return t->data_ptr();
  };
  const c10::cuda::CUDAGuard guard(device);
  // Rows of any tensor: 2-D ones keep their row stride, others are contiguous.
  auto in_rows = [&](const torch::Tensor& t) {
    return (t.dim() == 2 && t.stride(1) == 1) || t.is_contiguous() ? t : t.contiguous();
  };
  auto row_stride = [&](const torch::Tensor& t) { return t.dim() == 2 ? t.stride(0) : dim; };
  const torch::Tensor r = inplace ? residual : in_rows(residual);
  TORCH_CHECK(!inplace || (r.dim() == 2 && r.stride(1) == 1) || r.is_contiguous(),
              "an in-place residual must have contiguous rows");
  a.residual = r.data_ptr();
  a.residual_stride = row_stride(r);
  torch::Tensor yc, gc, h, out = residual;
  if (y) {
    TORCH_CHECK(y->is_cuda() && y->device() == device && y->sizes() == residual.sizes(),
                "y must have residual's shape and device");
    yc = in_rows(*y);
    a.y = yc.data_ptr();
    a.y_stride = row_stride(yc);
  }
  if (gate) {
    TORCH_CHECK(gate->is_cuda() && gate->device() == device && gate->scalar_type() == type,
                "gate must have y's type and device");
    const bool channel = gate->dim() == 1 && gate->size(0) == dim;
    const bool full = gate->sizes() == residual.sizes();
    bool row = !full && gate->dim() == residual.dim() && gate->size(-1) == 1;
    for (int64_t i = 0; row && i + 1 < residual.dim(); ++i) row = gate->size(i) == residual.size(i);
    TORCH_CHECK(channel || full || row, "gate must be [dim], [..., 1] or [..., dim]");
    gc = full ? in_rows(*gate) : gate->contiguous();
    a.gate = gc.data_ptr();
    a.gate_column_stride = row ? 0 : 1;
    a.gate_stride = full ? row_stride(gc) : row ? 1 : 0;
  }
  a.post_weight = weight(post_weight, "post_weight");
  a.post_bias = weight(post_bias, "post_bias");
  a.pre_weight = weight(pre_weight, "pre_weight");
  a.pre_bias = weight(pre_bias, "pre_bias");
  // Without y and with a scale of 1 the residual stays what it is.
  // Two small outputs of one type come from one allocation.
  OptTensor result;
  const int64_t bytes = (residual.numel() * 2 + 15) / 16 * 16;
  if ((y || residual_scale != 1.0) && !inplace && pre_weight && residual.scalar_type() == type &&
      bytes <= (1 << 18)) {
    const torch::Tensor whole = torch::empty({2 * bytes}, residual.options().dtype(torch::kUInt8));
    out = part_of(whole, type, 0, residual.sizes());
    result = part_of(whole, type, bytes, residual.sizes());
  }
  if (y || residual_scale != 1.0) {
    if (!inplace && !result) out = torch::empty(residual.sizes(), residual.options());
    a.residual_out = out.data_ptr();
    a.residual_out_stride = inplace ? row_stride(r) : dim;
  }
  if (pre_weight) {
    if (!result) result = torch::empty(residual.sizes(), pre_weight->options());
    a.h = result->data_ptr();
    a.h_stride = dim;
  }
  a.rows = static_cast<int>(rows);
  a.dim = static_cast<int>(dim);
  a.kind = static_cast<dk_norm_kind>(kind);
  a.act = static_cast<dk_gate_act>(act);
  a.residual_scale = static_cast<float>(residual_scale);
  a.block_scale = static_cast<float>(block_scale);
  a.eps = static_cast<float>(eps);
  check_status(dk_block_norm(&a, at::cuda::getCurrentCUDAStream().stream()), "block_norm");
  return {out, result};
}

// ---------------------------------------------------------------------------
// A prompt's step: products of many rows, their gradients, rotary positions, the
// cache read back.
// ---------------------------------------------------------------------------
// Rows of `width` values of a tensor of any shape: a 2-D one whose rows the
// kernels can read where they lie, else a copy of it (its rows a multiple of 8
// values apart).
torch::Tensor in_rows(const torch::Tensor& t, int64_t width) {
  const int64_t rows = t.numel() / std::max<int64_t>(width, 1);
  torch::Tensor r = t.dim() == 2 ? t : t.reshape({rows, width});
  if (aligned16(r) && (width == 1 || r.stride(1) == 1) && (rows <= 1 || (r.stride(0) % 8 == 0 && r.stride(0) >= width))) return r;
  const torch::Tensor home = torch::empty({rows, (width + 7) / 8 * 8}, t.options()).narrow(1, 0, width);
  home.copy_(r);
  return home;
}

int64_t row_stride(const torch::Tensor& r) { return r.size(0) > 1 ? r.stride(0) : (r.size(1) + 7) / 8 * 8; }

// A pair of weights, checked; re-homed where it does not begin on 16 bytes.
struct Weights {
  torch::Tensor packed, scales;
  int64_t M, K;

  Weights(const torch::Tensor& p, const torch::Tensor& s, const torch::Tensor& x) : packed(p), scales(s) {
    TORCH_CHECK(p.is_cuda() && s.is_cuda() && x.is_cuda(), "packed, scales, and x must be CUDA tensors");
    TORCH_CHECK(p.scalar_type() == torch::kInt32, "packed must be int32 (uint32 bit pattern)");
    TORCH_CHECK(s.scalar_type() == torch::kFloat16, "scales must be fp16");
    TORCH_CHECK(p.dim() == 2 && s.dim() == 2, "packed [M,K/8], scales [M,K/128]");
    TORCH_CHECK(p.is_contiguous() && s.is_contiguous(), "packed and scales must be contiguous");
    TORCH_CHECK(p.device() == x.device() && s.device() == x.device(), "packed, scales, and x must be on the same device");
    M = p.size(0);
    K = p.size(1) * DK_NIBBLES_PER_WORD;
    TORCH_CHECK(K >= DK_GROUP_SIZE && K % DK_GROUP_SIZE == 0, "K must be divisible by group size 128");
    TORCH_CHECK(s.size(0) == M && s.size(1) == K / DK_GROUP_SIZE, "scales shape must be [M, K/128]");
    TORCH_CHECK(M <= INT32_MAX && K <= INT32_MAX, "dimensions must fit in int32");
    if (!aligned16(packed)) packed = packed.clone();
  }
  const int32_t* words() const { return packed.data_ptr<int32_t>(); }
  const uint16_t* factors() const { return reinterpret_cast<const uint16_t*>(scales.data_ptr<at::Half>()); }
};

// x of [..., width]: its other dimensions, with `last` behind them.
std::vector<int64_t> shape_with(const torch::Tensor& x, int64_t last) {
  std::vector<int64_t> shape = x.sizes().vec();
  shape.back() = last;
  return shape;
}

void check_rows(const torch::Tensor& x, int64_t width, const char* what) {
  TORCH_CHECK(x.dim() >= 1 && x.size(-1) == width, what, " must be [..., " + std::to_string(width) + "]");
  TORCH_CHECK(x.numel() / std::max<int64_t>(width, 1) <= INT32_MAX, what, " has too many rows");
}

dk_mlp_act mlp_act(int act) {
  TORCH_CHECK(act == DK_MLP_SILU || act == DK_MLP_GELU, "unknown activation");
  return static_cast<dk_mlp_act>(act);
}

// A kernel wrote over a tensor of the caller's: a graph that saved what stood there
// learns of it.
void written(const torch::Tensor& t) {
  if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

// Whether two tensors have a byte in common, for any strides.  With D the distance
// of a value of a from a value of b they do where -size_a < D < size_b for some choice
// of indices: D is a sum of index * stride, tried from the largest stride on with
// only those indices from which the smaller ones can still reach.  Strides that nest,
// as those of slices do, leave an index or two each; a search that would go on for
// long counts as a byte in common.
struct Strides {
  std::vector<std::array<int64_t, 5>> of;  // stride, its lowest and highest index, what it and the smaller ones reach
  int64_t low, high;                       // of D
  int tries = 1 << 14;

  // A tensor's values, contiguous ones taken as one; returns their bytes.
  int64_t add(const torch::Tensor& t, bool minus) {
    std::vector<std::pair<int64_t, int64_t>> dims;
    for (int64_t i = 0; i < t.dim(); ++i)
      if (t.size(i) > 1 && t.stride(i) != 0) dims.emplace_back(t.stride(i) * t.element_size(), t.size(i));
    std::sort(dims.begin(), dims.end());
    int64_t run = t.element_size();
    for (const auto& [stride, size] : dims) {
      if (stride == run) {
        run *= size;
        continue;
      }
      const auto at = std::find_if(of.begin(), of.end(), [s = stride](const auto& o) { return o[0] == s; });
      auto& mine = at != of.end() ? *at : of.emplace_back(std::array<int64_t, 5>{stride, 0, 0, 0, 0});
      mine[minus ? 1 : 2] += minus ? 1 - size : size - 1;
    }
    return run;
  }
  bool meet(size_t i, int64_t distance) {
    if (i == of.size()) return distance > low && distance < high;
    if (--tries < 0) return true;
    const auto [stride, first, last, below, above] = of[i];
    const int64_t rest_below = i + 1 < of.size() ? of[i + 1][3] : 0, rest_above = i + 1 < of.size() ? of[i + 1][4] : 0;
    // low < distance + n * stride + rest < high
    auto down = [](int64_t a, int64_t b) { return a >= 0 ? a / b : -((b - 1 - a) / b); };
    const int64_t from = std::max(first, down(low - distance - rest_above, stride) + 1);
    const int64_t to = std::min(last, -down(-(high - distance - rest_below), stride) - 1);
    for (int64_t n = from; n <= to; ++n)
      if (meet(i + 1, distance + n * stride)) return true;
    return false;
  }
};

bool shares_memory(const torch::Tensor& a, const torch::Tensor& b) {
  if (a.numel() == 0 || b.numel() == 0) return false;
  const int64_t distance = static_cast<int64_t>(reinterpret_cast<intptr_t>(a.data_ptr()) - reinterpret_cast<intptr_t>(b.data_ptr()));
  auto reach = [](const torch::Tensor& t) {  // from the first byte to behind the last
    int64_t values = 1;
    for (int64_t i = 0; i < t.dim(); ++i) values += (t.size(i) - 1) * t.stride(i);
    return values * t.element_size();
  };
  if (distance >= reach(b) || -distance >= reach(a)) return false;
  Strides s;
  s.high = s.add(b, true);
  s.low = -s.add(a, false);
  std::sort(s.of.begin(), s.of.end(), [](const auto& p, const auto& q) { return p[0] > q[0]; });
  int64_t below = 0, above = 0;
  for (size_t i = s.of.size(); i-- > 0;) {
    s.of[i][3] = below += s.of[i][0] * s.of[i][1];
    s.of[i][4] = above += s.of[i][0] * s.of[i][2];
  }
  return s.meet(0, distance);
}

// Forward-mode derivatives would be lost (or, of tensors written over, go stale).
void check_no_tangent(std::initializer_list<const torch::Tensor*> tensors) {
  for (const torch::Tensor* t : tensors)
    TORCH_CHECK(!t || !t->defined() || !t->_fw_grad(0).defined(), "forward-mode derivatives are not supported");
}
// What is written over keeps no history: a gradient through it would be that of what
// stood there.
void check_no_history(const OptTensor& out) {
  TORCH_CHECK(!out || !torch::GradMode::is_enabled() || !out->requires_grad(),
              "out takes no part in a gradient: give one that requires none, or call under torch.no_grad()");
}
const torch::Tensor* if_any(const OptTensor& t) { return t ? &*t : nullptr; }

// What a kernel writes is nothing of what it reads.
void check_apart(const torch::Tensor& out, const char* what, std::initializer_list<const torch::Tensor*> inputs) {
  for (const torch::Tensor* in : inputs)
    TORCH_CHECK(!in || !shares_memory(out, *in), what, " may not overlap the call's inputs");
}

// An output given by the caller: contiguous rows of any stride, or a new one.
torch::Tensor output(const OptTensor& out, const std::vector<int64_t>& shape, const torch::Tensor& x,
                     std::initializer_list<const torch::Tensor*> others) {
  if (!out) return torch::empty(shape, x.options());
  TORCH_CHECK(out->device() == x.device() && out->scalar_type() == x.scalar_type() && out->sizes() == c10::IntArrayRef(shape),
              "out must have the product's shape and x's type and device");
  TORCH_CHECK(out->is_contiguous() || (out->dim() == 2 && out->stride(1) == 1 && out->stride(0) >= out->size(1)),
              "out must have contiguous rows");
  check_apart(*out, "out", {&x});
  check_apart(*out, "out", others);
  return *out;
}

std::tuple<torch::Tensor, OptTensor, OptTensor> w4a16_gemm(torch::Tensor packed, torch::Tensor scales, OptTensor packed2,
                                                           OptTensor scales2, torch::Tensor x, int act, bool keep,
                                                           OptTensor out) {
  check_no_tangent({&x, &scales, if_any(scales2), if_any(out)});
  check_no_history(out);
  const Weights w(packed, scales, x);
  dk_gemm_args a{};
  a.dtype = half_type(x, "x");
  a.act = mlp_act(act);
  check_rows(x, w.K, "x");
  const c10::cuda::CUDAGuard guard(x.device());
  std::optional<Weights> w2;
  if (packed2) {
    w2.emplace(*packed2, *scales2, x);
    TORCH_CHECK(w2->M == w.M && w2->K == w.K, "gate and up must have the same shape");
    a.packed2 = w2->words();
    a.scales2 = w2->factors();
  }
  const torch::Tensor xr = in_rows(x, w.K);
  const std::vector<int64_t> shape = shape_with(x, w.M);
  torch::Tensor y = output(out, shape, x, {&packed, &scales, if_any(packed2), if_any(scales2)});
  OptTensor g, u;
  if (keep) {  // kept for the gradient, whose product wants rows a multiple of 8 apart
    const int64_t wide = (w.M + 7) / 8 * 8;
    const torch::Tensor whole = torch::empty({2, xr.size(0), wide}, x.options());
    g = whole[0].narrow(1, 0, w.M);
    u = whole[1].narrow(1, 0, w.M);
    a.gate_out = g->data_ptr();
    a.up_out = u->data_ptr();
    a.ldk = wide;
  }
  a.packed = w.words();
  a.scales = w.factors();
  a.x = xr.data_ptr();
  a.ldx = row_stride(xr);
  a.y = y.data_ptr();
  a.ldy = y.dim() == 2 && y.size(0) > 1 ? y.stride(0) : w.M;
  a.rows = static_cast<int>(xr.size(0));
  a.M = static_cast<int>(w.M);
  a.K = static_cast<int>(w.K);
  torch::Tensor workspace;
  if (const size_t need = dk_w4a16_gemm_workspace_bytes(a.rows, a.K, packed2 ? 2 : 1, a.dtype)) {
    workspace = torch::empty({static_cast<int64_t>(need)}, x.options().dtype(torch::kUInt8));
    a.workspace = workspace.data_ptr();
    a.workspace_bytes = need;
  }
  check_status(dk_w4a16_gemm(&a, at::cuda::getCurrentCUDAStream().stream()), "w4a16_gemm");
  if (out) written(y);
  return {y, g, u};
}

torch::Tensor w4a16_gemm_t(torch::Tensor packed, torch::Tensor scales, OptTensor packed2, OptTensor scales2,
                           torch::Tensor g, OptTensor g2, OptTensor out) {
  check_no_tangent({&g, &scales, if_any(g2), if_any(scales2), if_any(out)});
  check_no_history(out);
  const Weights w(packed, scales, g);
  dk_gemm_t_args a{};
  a.dtype = half_type(g, "g");
  check_rows(g, w.M, "g");
  const c10::cuda::CUDAGuard guard(g.device());
  if (w.M == 0) return output(out, shape_with(g, w.K), g, {}).zero_();
  torch::Tensor gr = in_rows(g, w.M), gr2;
  std::optional<Weights> w2;
  if (packed2) {
    w2.emplace(*packed2, *scales2, g);
    TORCH_CHECK(w2->M == w.M && w2->K == w.K, "gate and up must have the same shape");
    TORCH_CHECK(g2 && g2->sizes() == g.sizes() && g2->scalar_type() == g.scalar_type() && g2->device() == g.device(),
                "g2 must have g's shape, type and device");
    gr2 = in_rows(*g2, w.M);
    if (row_stride(gr2) != row_stride(gr)) {
      gr = in_rows(gr.contiguous(), w.M);
      gr2 = in_rows(gr2.contiguous(), w.M);
    }
    a.packed2 = w2->words();
    a.scales2 = w2->factors();
    a.g2 = gr2.data_ptr();
  }
  torch::Tensor dx = output(out, shape_with(g, w.K), g, {&packed, &scales, if_any(packed2), if_any(scales2), if_any(g2)});
  a.packed = w.words();
  a.scales = w.factors();
  a.g = gr.data_ptr();
  a.ldg = row_stride(gr);
  a.dx = dx.data_ptr();
  a.lddx = dx.dim() == 2 && dx.size(0) > 1 ? dx.stride(0) : w.K;
  a.rows = static_cast<int>(gr.size(0));
  a.M = static_cast<int>(w.M);
  a.K = static_cast<int>(w.K);
  check_status(dk_w4a16_gemm_t(&a, at::cuda::getCurrentCUDAStream().stream()), "w4a16_gemm_t");
  if (out) written(dx);
  return dx;
}

std::tuple<torch::Tensor, torch::Tensor> gated_grad(torch::Tensor dh, torch::Tensor g, torch::Tensor u, int act) {
  TORCH_CHECK(dh.is_cuda() && g.is_cuda() && u.is_cuda() && g.device() == dh.device() && u.device() == dh.device(),
              "dh, g and u must be CUDA tensors of one device");
  const dk_dtype type = half_type(dh, "dh");
  TORCH_CHECK(g.dim() == 2 && u.sizes() == g.sizes() && g.scalar_type() == dh.scalar_type() &&
                  u.scalar_type() == dh.scalar_type() && dh.numel() == g.numel(),
              "g and u must be [rows, M] with dh's type");
  TORCH_CHECK(g.stride(1) == 1 && u.strides() == g.strides(), "g and u must have contiguous rows and the same strides");
  const int64_t rows = g.size(0), M = g.size(1);
  TORCH_CHECK(rows <= INT32_MAX && M <= INT32_MAX, "dimensions must fit in int32");
  const c10::cuda::CUDAGuard guard(dh.device());
  const torch::Tensor d = in_rows(dh, M);
  const int64_t wide = (M + 7) / 8 * 8;
  const torch::Tensor whole = torch::empty({2, rows, wide}, dh.options());
  const torch::Tensor dg = whole[0].narrow(1, 0, M), du = whole[1].narrow(1, 0, M);
  check_status(dk_gated_grad(d.data_ptr(), g.data_ptr(), u.data_ptr(), dg.data_ptr(), du.data_ptr(), static_cast<int>(rows),
                             static_cast<int>(M), row_stride(d), row_stride(g), wide, type, mlp_act(act),
                             at::cuda::getCurrentCUDAStream().stream()),
               "gated_grad");
  return {dg, du};
}

std::tuple<torch::Tensor, OptTensor> rotary(torch::Tensor q, OptTensor k, torch::Tensor positions, torch::Tensor frequency,
                                            std::optional<std::vector<int64_t>> sections, bool paired, bool inverse,
                                            bool inplace) {
  check_no_tangent({&q, if_any(k), &frequency});
  TORCH_CHECK(q.is_cuda(), "q must be a CUDA tensor");
  TORCH_CHECK(q.dim() == 3, "q must be [tokens, q_heads, head_dim]");
  const torch::Device device = q.device();
  const int64_t tokens = q.size(0), dim = q.size(2);
  TORCH_CHECK(q.scalar_type() == torch::kFloat16 || q.scalar_type() == torch::kBFloat16 || q.scalar_type() == torch::kFloat32,
              "q must be fp16, bf16 or fp32");
  TORCH_CHECK(tokens <= INT32_MAX && q.size(1) >= 1 && q.size(1) < (1 << 20), "q must have 1 to 2^20 heads and less than 2^31 tokens");
  TORCH_CHECK(dim >= 2 && dim <= DK_ROTARY_MAX_DIM, "head_dim must be 2 to " + std::to_string(DK_ROTARY_MAX_DIM));
  if (k) {
    TORCH_CHECK(k->is_cuda() && k->device() == device && k->scalar_type() == q.scalar_type(), "k must have q's type and device");
    TORCH_CHECK(k->dim() == 3 && k->size(0) == tokens && k->size(2) == dim && k->size(1) >= 1 && k->size(1) < (1 << 20),
                "k must be [tokens, kv_heads, head_dim]");
  }
  TORCH_CHECK(frequency.is_cuda() && frequency.device() == device && frequency.scalar_type() == torch::kFloat32 &&
                  frequency.dim() == 1 && frequency.is_contiguous(),
              "frequency must be contiguous fp32 [pairs] on q's device");
  const int64_t pairs = frequency.size(0);
  TORCH_CHECK(pairs >= 1 && 2 * pairs <= dim, "frequency must have 1 to head_dim / 2 values");
  TORCH_CHECK(positions.is_cuda() && positions.device() == device, "positions must be on q's device");
  TORCH_CHECK(positions.scalar_type() == torch::kInt32 || positions.scalar_type() == torch::kInt64, "positions must be int32 or int64");
  TORCH_CHECK((positions.dim() == 1 || positions.dim() == 2) && positions.size(-1) == tokens,
              "positions must be [tokens] or [axes, tokens]");
  dk_rotary_args a{};
  const int64_t axes = positions.dim() == 2 ? positions.size(0) : 1;
  TORCH_CHECK(axes >= 1 && axes <= DK_ROTARY_MAX_AXES, "positions must have 1 to " + std::to_string(DK_ROTARY_MAX_AXES) + " axes");
  TORCH_CHECK(sections || axes == 1, "several axes need sections");
  if (sections) {
    TORCH_CHECK(static_cast<int64_t>(sections->size()) == axes, "sections must have a number of pairs for each axis");
    int64_t end = 0;
    for (int64_t i = 0; i < axes; ++i) {
      TORCH_CHECK((*sections)[i] >= 0 && (*sections)[i] <= pairs, "sections must be numbers of pairs");
      a.section_end[i] = static_cast<int>(end += (*sections)[i]);
    }
    TORCH_CHECK(end == pairs, "sections must add up to frequency's length");
  } else {
    a.section_end[0] = static_cast<int>(pairs);
  }
  const c10::cuda::CUDAGuard guard(device);
  const torch::Tensor at = positions.stride(-1) == 1 || tokens <= 1 ? positions : positions.contiguous();
  // Two small outputs come from one allocation.
  torch::Tensor whole;
  const int64_t size = static_cast<int64_t>(q.element_size()), q_bytes = (q.numel() * size + 15) / 16 * 16;
  if (k && !inplace && q_bytes + k->numel() * size <= (1 << 22))
    whole = torch::empty({q_bytes + k->numel() * size}, q.options().dtype(torch::kUInt8));
  auto place = [&](const torch::Tensor& t, int64_t byte, const void*& in, void*& out, int64_t& it, int64_t& ih, int64_t& ot, int64_t& oh) {
    if (inplace) {
      TORCH_CHECK(t.stride(2) == 1, "q and k that are turned in place must have contiguous heads");
      for (int64_t i = 0; i < 2; ++i)
        TORCH_CHECK(t.size(i) == 1 || t.stride(i) >= dim, "q and k that are turned in place may not overlap themselves");
      TORCH_CHECK(t.size(0) <= 1 || t.size(1) == 1 || t.stride(0) >= (t.size(1) - 1) * t.stride(1) + dim ||
                      t.stride(1) >= (t.size(0) - 1) * t.stride(0) + dim,
                  "q and k that are turned in place may not overlap themselves");
    }
    const torch::Tensor from = t.stride(2) == 1 ? t : t.contiguous();
    const torch::Tensor to = inplace ? t : whole.defined() ? part_of(whole, t.scalar_type(), byte, t.sizes()) : torch::empty(t.sizes(), t.options());
    in = from.data_ptr();
    out = to.data_ptr();
    it = from.stride(0), ih = from.stride(1), ot = to.stride(0), oh = to.stride(1);
    return std::make_pair(from, to);
  };
  const auto qs = place(q, 0, a.q, a.q_out, a.q_token_stride, a.q_head_stride, a.q_out_token_stride, a.q_out_head_stride);
  std::pair<torch::Tensor, torch::Tensor> ks;
  if (k) {
    ks = place(*k, q_bytes, a.k, a.k_out, a.k_token_stride, a.k_head_stride, a.k_out_token_stride, a.k_out_head_stride);
    TORCH_CHECK(!inplace || !shares_memory(q, *k), "q and k that are turned in place may not overlap each other");
    if (inplace) check_apart(*k, "k", {&positions, &frequency});
    a.kv_heads = static_cast<int>(k->size(1));
  }
  if (inplace) check_apart(q, "q", {&positions, &frequency});
  a.positions = at.data_ptr();
  a.positions_64 = at.scalar_type() == torch::kInt64;
  a.position_stride = at.dim() == 2 ? at.stride(0) : 0;
  a.frequency = frequency.data_ptr<float>();
  a.tokens = static_cast<int>(tokens);
  a.q_heads = static_cast<int>(q.size(1));
  a.head_dim = static_cast<int>(dim);
  a.pairs = static_cast<int>(pairs);
  a.axes = static_cast<int>(axes);
  a.paired = paired;
  a.inverse = inverse;
  a.dtype = q.scalar_type() == torch::kFloat32 ? DK_FP32 : half_type(q, "q");
  check_status(dk_rotary(&a, at::cuda::getCurrentCUDAStream().stream()), "rotary");
  if (inplace) {
    written(q);
    if (k) written(*k);
  }
  return {qs.second, k ? OptTensor(ks.second) : OptTensor()};
}

std::tuple<torch::Tensor, torch::Tensor> cache_read(const Cache8& cache, torch::Tensor block_table, torch::Tensor lengths,
                                                    torch::Tensor starts, int64_t tokens, torch::ScalarType type, OptTensor k,
                                                    OptTensor v) {
  check_no_tangent({if_any(k), if_any(v)});
  check_no_history(k);
  check_no_history(v);
  const torch::Device device = cache.k.device();
  TORCH_CHECK(lengths.dim() == 1, "lengths must be [requests]");
  const int64_t n = lengths.size(0);
  TORCH_CHECK(n <= INT32_MAX - 1, "too many requests");
  TORCH_CHECK(tokens >= 0 && tokens <= INT32_MAX, "tokens out of range");
  check_ints(lengths, torch::kInt32, n, device, "lengths");
  check_ints(starts, torch::kInt32, n + 1, device, "starts");
  check_table(block_table, n, device);
  TORCH_CHECK(type == torch::kFloat16 || type == torch::kBFloat16, "dtype must be fp16 or bf16");
  const c10::cuda::CUDAGuard guard(device);
  const std::vector<int64_t> shape = {tokens, cache.c.kv_heads, cache.c.head_dim};
  // Two small outputs come from one allocation.
  torch::Tensor whole;
  const int64_t bytes = tokens * cache.c.kv_heads * cache.c.head_dim * 2;  // a multiple of 16
  if (!k && !v && bytes <= (1 << 21)) whole = torch::empty({2 * bytes}, cache.k.options().dtype(torch::kUInt8));
  auto given = [&](const OptTensor& t, const char* what) {
    if (!t && whole.defined()) return part_of(whole, type, *what == 'v' ? bytes : 0, shape);
    if (!t) return torch::empty(shape, cache.k.options().dtype(type));
    TORCH_CHECK(t->is_cuda() && t->device() == device && t->scalar_type() == type && t->sizes() == c10::IntArrayRef(shape),
                what, " must be [tokens, kv_heads, head_dim] of dtype on the cache's device");
    TORCH_CHECK(t->stride(2) == 1 && (t->size(1) == 1 || t->stride(1) == t->size(2)) &&
                    (tokens <= 1 || (t->stride(0) % 8 == 0 && t->stride(0) >= t->size(1) * t->size(2))) && aligned16(*t),
                what, " must have contiguous rows, a multiple of 8 values apart and 16-byte aligned");
    check_apart(*t, what, {&cache.k, &cache.v, &cache.k_scale, &cache.v_scale, &block_table, &lengths, &starts});
    return *t;
  };
  const torch::Tensor ko = given(k, "k"), vo = given(v, "v");
  TORCH_CHECK(!k || !v || !shares_memory(ko, vo), "k and v must be two tensors that do not overlap");
  dk_cache_read_args a{};
  a.cache = cache.c;
  a.block_table = block_table.data_ptr<int32_t>();
  a.max_blocks = static_cast<int>(block_table.size(1));
  a.table_stride = static_cast<int>(n > 1 ? block_table.stride(0) : block_table.size(1));
  a.lengths = lengths.data_ptr<int32_t>();
  a.starts = starts.data_ptr<int32_t>();
  a.requests = static_cast<int>(n);
  a.tokens = static_cast<int>(tokens);
  a.k = ko.data_ptr();
  a.v = vo.data_ptr();
  a.k_token_stride = tokens > 1 ? ko.stride(0) : 0;
  a.v_token_stride = tokens > 1 ? vo.stride(0) : 0;
  a.dtype = type == torch::kFloat16 ? DK_FP16 : DK_BF16;
  check_status(dk_cache_read(&a, at::cuda::getCurrentCUDAStream().stream()), "cache_read");
  if (k) written(*k);
  if (v) written(*v);
  return {ko, vo};
}

// ---------------------------------------------------------------------------
// Gradients.  The linear operators are each other's gradients (a turning's is the
// turning back), so they may be differentiated any number of times.
// ---------------------------------------------------------------------------
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

bool wants_grad(const torch::Tensor& x, const torch::Tensor& scales) {
  if (!torch::GradMode::is_enabled()) return false;
  TORCH_CHECK(!scales.requires_grad(), "the weights are frozen: scales must not require a gradient");
  return x.requires_grad();
}

torch::Tensor linear(bool transposed, const torch::Tensor& packed, const torch::Tensor& scales, const torch::Tensor& x, OptTensor out);

struct Linear : torch::autograd::Function<Linear> {
  static torch::Tensor forward(AutogradContext* ctx, torch::Tensor x, torch::Tensor packed, torch::Tensor scales, bool transposed) {
    ctx->save_for_backward({packed, scales});
    ctx->saved_data["transposed"] = transposed;
    const at::AutoDispatchBelowADInplaceOrView below;
    return transposed ? w4a16_gemm_t(packed, scales, {}, {}, x, {}, {}) : std::get<0>(w4a16_gemm(packed, scales, {}, {}, x, 0, false, {}));
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const variable_list saved = ctx->get_saved_variables();
    return {linear(!ctx->saved_data["transposed"].toBool(), saved[0], saved[1], grads[0], {}), {}, {}, {}};
  }
};

torch::Tensor linear(bool transposed, const torch::Tensor& packed, const torch::Tensor& scales, const torch::Tensor& x, OptTensor out) {
  if (wants_grad(x, scales)) {
    TORCH_CHECK(!out, "out takes no part in a gradient: call without it or under torch.no_grad()");
    return Linear::apply(x, packed, scales, transposed);
  }
  return transposed ? w4a16_gemm_t(packed, scales, {}, {}, x, {}, out) : std::get<0>(w4a16_gemm(packed, scales, {}, {}, x, 0, false, out));
}

using Pair = std::tuple<torch::Tensor, OptTensor>;
Pair turn(torch::Tensor q, OptTensor k, torch::Tensor positions, torch::Tensor frequency, std::optional<std::vector<int64_t>> sections,
          bool paired, bool inverse, bool inplace);

struct Turn : torch::autograd::Function<Turn> {
  static variable_list forward(AutogradContext* ctx, torch::Tensor q, OptTensor k, torch::Tensor positions, torch::Tensor frequency,
                               std::optional<std::vector<int64_t>> sections, bool paired, bool inverse) {
    ctx->save_for_backward({positions, frequency});
    ctx->saved_data["sections"] = sections;
    ctx->saved_data["paired"] = paired;
    ctx->saved_data["inverse"] = inverse;
    const at::AutoDispatchBelowADInplaceOrView below;
    const Pair both = rotary(q, k, positions, frequency, sections, paired, inverse, false);
    return k ? variable_list{std::get<0>(both), *std::get<1>(both)} : variable_list{std::get<0>(both)};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const variable_list saved = ctx->get_saved_variables();
    std::optional<std::vector<int64_t>> sections;
    if (!ctx->saved_data["sections"].isNone()) sections = ctx->saved_data["sections"].toIntVector();
    const Pair both = turn(grads[0], grads.size() > 1 ? OptTensor(grads[1]) : OptTensor(), saved[0], saved[1], sections,
                           ctx->saved_data["paired"].toBool(), !ctx->saved_data["inverse"].toBool(), false);
    return {std::get<0>(both), grads.size() > 1 ? *std::get<1>(both) : torch::Tensor(), {}, {}, {}, {}, {}};
  }
};

Pair turn(torch::Tensor q, OptTensor k, torch::Tensor positions, torch::Tensor frequency, std::optional<std::vector<int64_t>> sections,
          bool paired, bool inverse, bool inplace) {
  if (torch::GradMode::is_enabled()) {
    TORCH_CHECK(!frequency.requires_grad(), "frequency must not require a gradient");
    if (q.requires_grad() || (k && k->requires_grad())) {
      TORCH_CHECK(!inplace, "q and k that require a gradient are not turned in place");
      const variable_list out = Turn::apply(q, k, positions, frequency, sections, paired, inverse);
      return {out[0], k ? OptTensor(out[1]) : OptTensor()};
    }
  }
  return rotary(q, k, positions, frequency, sections, paired, inverse, inplace);
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  m.def("w4a16_gemv", &w4a16_gemv, "W4A16 GEMV", py::arg("packed"), py::arg("scales"),
        py::arg("x"), py::arg("version") = 5, py::arg("split_k") = 4,
        py::arg("reuse_weights") = false, py::arg("warps_per_row") = 1);
  m.def("w4a16_gemv_out", &w4a16_gemv_out, "W4A16 GEMV into a caller-provided y",
        py::arg("packed"), py::arg("scales"), py::arg("x"), py::arg("y"), py::arg("version") = 5,
        py::arg("split_k") = 4, py::arg("reuse_weights") = false, py::arg("warps_per_row") = 1,
        py::arg("pdl") = false);
  m.def("workspace_bytes", &workspace_bytes, "Workspace bytes for a GEMV", py::arg("M"),
        py::arg("K"), py::arg("B"), py::arg("version") = 5, py::arg("split_k") = 4,
        py::arg("reuse_weights") = false);
  m.def("d2d_copy", &d2d_copy, "Aligned device-to-device copy", py::arg("src"), py::arg("dst"));
  m.def("stream_read", &stream_read, "Read-only STREAM sum-reduction (one float partial per block)",
        py::arg("src"), py::arg("partials"));
  m.def("stream_write", &stream_write, "Write-only STREAM fill", py::arg("dst"));
  m.def("stream_recommended_blocks", &stream_recommended_blocks,
        "Block count used by STREAM probes");
  m.def("last_kernel_stamp", &last_kernel_stamp,
        "Stage stamp written by the GEMV that actually launched");
  m.def("device_error", &device_error, "Device-side error word (1 = bounded wait timed out)",
        py::arg("clear") = false);
  m.def("quantize_pack", &quantize_pack, "GPU quantize_and_pack (bit-exact)", py::arg("weight"),
        py::arg("torch_cuda_scale") = false);
  m.def("unpack_to_int", &unpack_to_int, "GPU unpack_to_int", py::arg("packed"));
  m.def("dequantize", &dequantize, "GPU dequantize to fp32", py::arg("packed"), py::arg("scales"));
  py::class_<Cache8>(m, "Cache8")
      .def(py::init<torch::Tensor, torch::Tensor, torch::Tensor, torch::Tensor>(), py::arg("k"),
           py::arg("v"), py::arg("k_scale"), py::arg("v_scale"));
  m.def("cache_plan", &cache_plan, "Block tables and slot maps of a step", py::arg("held"),
        py::arg("fresh"), py::arg("block_table"), py::arg("free_blocks"), py::arg("ring"),
        py::arg("block_size"), py::arg("tokens"), py::arg("lengths") = py::none(),
        py::arg("starts") = py::none(), py::arg("slots") = py::none(),
        py::arg("ring_out") = py::none());
  m.def("cache_append", &cache_append, "New keys and values into a paged 8-bit cache", py::arg("k"),
        py::arg("v"), py::arg("slots"), py::arg("cache"));
  m.def("cache_attention", &cache_attention, "Attention over a paged 8-bit cache", py::arg("q"),
        py::arg("cache"), py::arg("block_table"), py::arg("lengths"), py::arg("starts") = py::none(),
        py::arg("scale") = py::none(), py::arg("causal") = true, py::arg("window") = 0,
        py::arg("out") = py::none(), py::arg("lse") = false);
  m.def("release_workspaces", &release_workspaces, "Drop the kept attention workspaces");
  m.def("block_norm", &block_norm, "Norms, gate and residual between two blocks",
        py::arg("residual"), py::arg("y"), py::arg("kind"), py::arg("post_weight"),
        py::arg("post_bias"), py::arg("gate"), py::arg("act"), py::arg("residual_scale"),
        py::arg("block_scale"), py::arg("pre_weight"), py::arg("pre_bias"), py::arg("eps"),
        py::arg("inplace"));
  m.def("linear", &linear, "A product of rows, or the transposed one; differentiable", py::arg("transposed"), py::arg("packed"), py::arg("scales"),
        py::arg("x"), py::arg("out") = py::none());
  m.def("w4a16_gemm", &w4a16_gemm, "Many rows through 4-bit weights, or through a gated pair", py::arg("packed"),
        py::arg("scales"), py::arg("packed2"), py::arg("scales2"), py::arg("x"), py::arg("act") = 0, py::arg("keep") = false,
        py::arg("out") = py::none());
  m.def("w4a16_gemm_t", &w4a16_gemm_t, "The transposed product", py::arg("packed"), py::arg("scales"), py::arg("packed2"),
        py::arg("scales2"), py::arg("g"), py::arg("g2") = py::none(), py::arg("out") = py::none());
  m.def("gated_grad", &gated_grad, "Gradients of a gated block's pre-activations", py::arg("dh"), py::arg("g"), py::arg("u"),
        py::arg("act"));
  m.def("rotary", &turn, "Rotary positions of queries and keys", py::arg("q"), py::arg("k"), py::arg("positions"),
        py::arg("frequency"), py::arg("sections"), py::arg("paired"), py::arg("inverse"), py::arg("inplace"));
  m.def("shares_memory", &shares_memory, "Whether two tensors have a byte in common", py::arg("a"), py::arg("b"));
  m.def("cache_read", &cache_read, "Keys and values of a paged 8-bit cache as rows", py::arg("cache"), py::arg("block_table"),
        py::arg("lengths"), py::arg("starts"), py::arg("tokens"), py::arg("dtype"), py::arg("k") = py::none(),
        py::arg("v") = py::none());
  m.def("version", []() { return std::string(dk_version()); });
}
