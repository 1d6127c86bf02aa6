// Attention of single tokens over the paged cache that also keeps what every key
// receives. The products are paged_decode.h's, whose waves here leave their scores
// (f32, log2 domain); once a row's maxima m and sums l are known,
//   W_j (+)= sum over the heads g of a kv group of exp2(s_gj - m_g) / l_g,
// one thread per four keys and kv head: no atomics. That is at the end of the same launch
// where one workgroup has all keys of a (sequence, kv head), and beside the fold
// where several have.
//
// What bounds it: memory, as the attention alone, and the launches of small steps.
// Next to 4 D bytes of a key's K and V (bf16) are 4 G of scores, written and read
// again out of the caches, and 8 of its weight. Measured with 32/8 heads of 128, and
// with scores weighed in a launch of their own, a key a thread: one row of 217 keys
// 8.3 us (10.0 in two launches); 64 of 1500 to 4096 180 us, 4.2 TB/s (187; the
// attention alone 171; a key a thread in this launch 208); 256 of 30 to 1000, 8/4
// heads of 256, 128 (132); 16 of 8000 to 16000 e4m3 keys, 64/8 heads of 64, 47 and 15
// beside the fold (46, 5 and 16), which reads 65 MB of scores at 4.3 TB/s.
#include "paged_decode.h"
#include "keys_common.h"
#include <torch/library.h>

namespace kaito {

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
  a.scores = scores.data_ptr<float>();
  a.key_weights = key_weights.data_ptr<float>();
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
}

}  // namespace kaito

TORCH_LIBRARY_FRAGMENT(kaito, m) {
  m.def("paged_attention_weights(Tensor(a!) out, Tensor q, Tensor k_cache, Tensor v_cache, Tensor(b!) key_weights, Tensor block_tables, Tensor seq_lens, float scale, Tensor sinks) -> ()");
}
TORCH_LIBRARY_IMPL(kaito, CUDA, m) {
  m.impl("paged_attention_weights", &kaito::paged_attention_weights);
}
