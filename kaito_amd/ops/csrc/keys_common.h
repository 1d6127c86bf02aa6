// What the operators on weighted pages ("keys" group) check of their tensors.
#pragma once
#include <ATen/ATen.h>
#include <ATen/hip/HIPContext.h>
#include <ATen/hip/impl/HIPGuardImplMasqueradingAsCUDA.h>

namespace kaito {
namespace keys {

constexpr int PAGE = 16;            // keys of a page

// launches go to the tensors' device, on its current stream
using Guard = c10::hip::HIPGuardMasqueradingAsCUDA;

inline void check_int(const at::Tensor& t, const at::Tensor& on,
                      const char* name) {
  TORCH_CHECK(t.dtype() == at::kInt && t.is_contiguous() &&
              t.device() == on.device(), name, ": contiguous int32 on ",
              on.device());
}

// key_weights [NB, KH, 16] f32 and the tables that lead to them
inline void check_weights(const at::Tensor& key_weights,
                          const at::Tensor& block_tables) {
  TORCH_CHECK(key_weights.is_cuda() && key_weights.dtype() == at::kFloat &&
              key_weights.is_contiguous() && key_weights.dim() == 3 &&
              key_weights.size(2) == PAGE && key_weights.size(1) > 0 &&
              (uintptr_t)key_weights.data_ptr() % 16 == 0,
              "key_weights: contiguous f32 [pages, kv heads, 16] in 16 bytes");
  TORCH_CHECK(block_tables.dim() == 2 && block_tables.size(0) <= 65535 &&
              block_tables.size(1) <= (1 << 26),
              "block_tables: [sequences, pages]");
  check_int(block_tables, key_weights, "block_tables");
}

inline void check_pages(const at::Tensor& k_cache, const at::Tensor& v_cache,
                        const at::Tensor& key_weights) {
  const auto type = k_cache.dtype();
  TORCH_CHECK(k_cache.is_cuda() && k_cache.dim() == 4 &&
              k_cache.is_contiguous() && v_cache.is_contiguous() &&
              v_cache.sizes() == k_cache.sizes() && v_cache.dtype() == type &&
              k_cache.device() == v_cache.device() &&
              k_cache.device() == key_weights.device(),
              "caches: contiguous [pages, kv heads, 16, head_dim] of one type");
  TORCH_CHECK(k_cache.size(0) == key_weights.size(0) &&
              k_cache.size(1) == key_weights.size(1) &&
              k_cache.size(2) == PAGE, "key_weights are not these pages'");
  TORCH_CHECK((uintptr_t)k_cache.data_ptr() % 16 == 0 &&
              (uintptr_t)v_cache.data_ptr() % 16 == 0, "caches: 16-byte rows");
}

// query rows [T, QH, D] whose heads lie one behind another, and their output
inline void check_rows(const at::Tensor& out, const at::Tensor& q,
                       const at::Tensor& k_cache, const at::Tensor& sinks) {
  const int64_t D = k_cache.size(3);
  TORCH_CHECK(D == 64 || D == 128 || D == 256, "unsupported head_dim ", D);
  TORCH_CHECK(k_cache.dtype() == at::kBFloat16 || k_cache.dtype() == at::kByte,
              "pages: bf16 or e4m3 (uint8)");
  TORCH_CHECK(q.dtype() == at::kBFloat16 && q.dim() == 3 && q.size(2) == D &&
              q.size(1) > 0 && q.size(1) % k_cache.size(1) == 0 &&
              q.device() == k_cache.device(),
              "q: bf16 [rows, query heads, ", D, "]");
  TORCH_CHECK(q.stride(2) == 1 && q.stride(1) == D &&
              (q.size(0) < 2 || q.stride(0) % 8 == 0) &&
              (uintptr_t)q.data_ptr() % 16 == 0, "q: heads behind one another");
  TORCH_CHECK(out.is_contiguous() && out.sizes() == q.sizes() &&
              out.dtype() == q.dtype() && out.device() == q.device());
  TORCH_CHECK(sinks.numel() == 0 ||
              (sinks.dtype() == at::kFloat && sinks.is_contiguous() &&
               sinks.device() == q.device() && sinks.numel() == q.size(1)),
              "sinks: f32, one for each query head");
}

}  // namespace keys
}  // namespace kaito
