// Attention of single tokens over the paged cache that also keeps what every key
// receives. The products are paged_decode.h's, which here leaves its scores (f32,
// log2 domain) and every row's maximum m and 1 / sum; a second launch makes
//   W_j (+)= sum over the heads g of a kv group of exp2(s_gj - m_g) / l_g
// of them, one thread per key and kv head: no atomics. Next to the 4 D bytes of a
// key's K and V (bf16) the scores are 4 G bytes written and read.
#include "paged_decode.h"
#include "keys_common.h"
#include <torch/library.h>

namespace kaito {

namespace {

__global__ __launch_bounds__(256)
void row_weight_kernel(const DecodeArgs a, float* __restrict__ key_weights) {
  const int seq = blockIdx.y, kvh = blockIdx.x % a.KH;
  const int key = blockIdx.x / a.KH * 256 + threadIdx.x;
  const int len = a.len<false, true>(seq);
  if (key >= len) return;
  const int head = kvh * a.G;
  const int64_t row = (int64_t)seq * a.KH * a.G + head;
  const int page = a.block_tables[(int64_t)seq * a.max_blocks + key / BS];
  float* w = key_weights + ((int64_t)page * a.KH + kvh) * BS + key % BS;
  float sum = key + 1 < len ? *w : 0.f;
  for (int g = 0; g < a.G; g++) {
    const float s = a.scores[(row + g) * a.score_stride + key];
    const float2 st = a.stats[row + g];
    // what the attention gives no weight has none here
    if (s > -1e29f) sum += __builtin_amdgcn_exp2f(s - st.x) * st.y;
  }
  *w = sum;
}

}  // namespace

void paged_attention_weights(at::Tensor out, at::Tensor q, at::Tensor k_cache,
                             at::Tensor v_cache, at::Tensor key_weights,
                             at::Tensor block_tables, at::Tensor seq_lens,
                             double scale, at::Tensor sinks) {
  keys::check_weights(key_weights, block_tables);
  keys::check_pages(k_cache, v_cache, key_weights);
  keys::check_rows(out, q, k_cache, sinks);
  keys::check_int(seq_lens, q, "seq_lens");
  const int64_t T = q.size(0), QH = q.size(1), D = q.size(2);
  TORCH_CHECK(block_tables.size(0) == T && seq_lens.numel() == T);
  DecodeArgs a{};
  a.KH = k_cache.size(1);
  a.G = QH / a.KH;
  TORCH_CHECK(D == 128 ? a.G <= 8
              : D == 64 ? a.G == 1 || a.G == 2 || a.G == 4 || a.G == 8
                        : a.G == 1 || a.G == 2 || a.G == 4,
              "unsupported GQA group ", a.G, " of head_dim ", D);
  if (T == 0) return;
  a.max_blocks = block_tables.size(1);
  const keys::Guard guard(q.device());
  a.score_stride = ((int64_t)a.max_blocks * BS + KT - 1) / KT * KT;
  const auto f32 = q.options().dtype(at::kFloat);
  const at::Tensor scores = at::empty({T, QH, a.score_stride}, f32);
  const at::Tensor stats = at::empty({T, QH, 2}, f32);
  a.scores = scores.data_ptr<float>();
  a.stats = (float2*)stats.data_ptr<float>();
  a.out = (short*)out.data_ptr();
  a.q = (const short*)q.data_ptr();
  a.k = k_cache.data_ptr();
  a.v = v_cache.data_ptr();
  a.block_tables = block_tables.data_ptr<int>();
  a.seq_lens = seq_lens.data_ptr<int>();
  a.scale = (float)scale;
  a.q_stride = q.stride(0);
  if (sinks.numel() > 0) a.sinks = sinks.data_ptr<float>();
  const bool fp8 = k_cache.dtype() == at::kByte;
#define PW_DIM(D_)                                                            \
  if (D == D_) {                                                              \
    if (fp8) launch_paged_decode<D_, true, false, false, true>(a, out, T);    \
    else launch_paged_decode<D_, false, false, false, true>(a, out, T);       \
  }
  PW_DIM(64) PW_DIM(128) PW_DIM(256)
#undef PW_DIM
  if (a.max_blocks == 0) return;
  const int64_t blocks = ((int64_t)a.max_blocks * BS + 255) / 256;
  hipLaunchKernelGGL(row_weight_kernel, dim3(blocks * a.KH, T), dim3(256), 0,
                     at::hip::getCurrentHIPStream(), a,
                     key_weights.data_ptr<float>());
}

}  // namespace kaito

TORCH_LIBRARY_FRAGMENT(kaito, m) {
  m.def("paged_attention_weights(Tensor(a!) out, Tensor q, Tensor k_cache, Tensor v_cache, Tensor(b!) key_weights, Tensor block_tables, Tensor seq_lens, float scale, Tensor sinks) -> ()");
}
TORCH_LIBRARY_IMPL(kaito, CUDA, m) {
  m.impl("paged_attention_weights", &kaito::paged_attention_weights);
}
