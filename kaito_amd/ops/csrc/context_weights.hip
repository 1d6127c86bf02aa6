// Attention of chunks of new tokens over the paged cache that also keeps what
// every key receives:
//   p_ij = exp(s_ij - m_i) / l_i,   o_i = sum_j p_ij v_j   (flash_prefill.h)
//   W_j (+)= sum over the rows i that see key j, all heads of a kv group, of p_ij
// A key's weights need the rows' final maximum m and sum l, so that they are a
// second pass over the scores: the first leaves (m, 1 / l) of every row.
//
// The second pass keeps the keys and lets the rows go by, so that every key's sum
// has one owner: no atomics, the same bits every time. A workgroup is 4 waves x 64
// keys of a kv head. S^T = K Q^T on v_mfma_f32_32x32x16_bf16: the wave's K
// stays in registers as the first operand; query rows, flattened over the heads of
// the group (row = position * G + head), come in tiles of 64 through LDS, one
// tile ahead (swizzled as flash_prefill.h's K). A lane holds one row of a tile and
// 16 keys of every 32, so that m and 1 / l are per-lane scalars and a weight is a
// multiply-add, an exponential and a multiply-add into its key's sum.
#include "flash_prefill.h"
#include "keys_common.h"
#include <torch/library.h>

namespace kaito {

namespace {

using flash::hbf16x8;
using flash::f32x16;

constexpr int WKEYS = 64;           // keys of a wave
constexpr int KEYS = 4 * WKEYS;     // of a workgroup
constexpr int ROWS = 64;            // query rows of a tile

struct WeightArgs {
  const short* q;
  const void* k;
  float* key_weights;               // [NB, KH, 16]
  const float2* stats;              // [T, QH]
  const int* cu;
  const int* kv_lens;
  const int* block_tables;
  int64_t q_ts;
  int max_blocks, KH, G;
  unsigned div_g;                   // ceil(2^32 / G): rows / G by a product's high half
  float c;                          // scale * log2 e
};

// row / G, exact below 2^26 rows for G up to 64
KAITO_DEV int rows_over(const int row, const WeightArgs& a) {
  return a.G == 1 ? row : (int)__umulhi((unsigned)row, a.div_g);
}

template <int D, bool FP8>
__global__ __launch_bounds__(256, 2)
void key_weight_kernel(const WeightArgs a) {
  constexpr int KK = D / 16, CK = D / 8, COPIES = ROWS * CK / 256;
  const int seq = blockIdx.y;
  const int kvh = blockIdx.x % a.KH, key0 = blockIdx.x / a.KH * KEYS;
  const int tok0 = a.cu[seq], q_len = a.cu[seq + 1] - tok0;
  const int kv_len = min(a.kv_lens[seq], a.max_blocks * keys::PAGE);
  if (key0 >= kv_len || q_len <= 0) return;
  const int* bt = a.block_tables + (int64_t)seq * a.max_blocks;
  const int QH = a.KH * a.G, q_abs0 = kv_len - q_len;

  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int lr = lane & 31, h = lane >> 5;
  __shared__ __attribute__((aligned(128))) short lds[2][ROWS * D];

  // ---- this wave's keys
  const int wkey = key0 + wave * WKEYS;
  hbf16x8 kf[2][KK];
#pragma unroll
  for (int t = 0; t < 2; t++) {
    const int key = min(wkey + t * 32 + lr, kv_len - 1);
    const int64_t row =
        ((int64_t)bt[key / keys::PAGE] * a.KH + kvh) * keys::PAGE +
        key % keys::PAGE;
#pragma unroll
    for (int kk = 0; kk < KK; kk++) {
      const int64_t at = row * D + kk * 16 + h * 8;
      if constexpr (FP8) {
        float f[8];
        fp8x8_to_f32(*reinterpret_cast<const u8x8_t*>((const uint8_t*)a.k + at),
                     f);
#pragma unroll
        for (int e = 0; e < 8; e++) kf[t][kk][e] = (__bf16)f[e];
      } else {
        kf[t][kk] = *reinterpret_cast<const hbf16x8*>((const short*)a.k + at);
      }
    }
  }

  // ---- the rows that see one of the workgroup's keys
  const int rows = q_len * a.G;
  const int first = max(0, key0 - q_abs0) * a.G / ROWS * ROWS;
  auto stage = [&](const int r0, short* buf) {
#pragma unroll
    for (int j = 0; j < COPIES; j++) {
      const int s = j * 256 + tid, row = s / CK;
      const int R = min(r0 + row, rows - 1), pos = rows_over(R, a);
      const short* p = a.q + (int64_t)(tok0 + pos) * a.q_ts +
          (kvh * a.G + R - pos * a.G) * D + flash::swz_k<D>(row, s % CK) * 8;
      flash::lds_copy16(p, buf + (j * 256 + wave * 64) * 8);
    }
  };
  f32x16 sum[2];
#pragma unroll
  for (int t = 0; t < 2; t++)
#pragma unroll
    for (int i = 0; i < 16; i++) sum[t][i] = 0.f;

  stage(first, lds[0]);
  __syncthreads();
  int cur = 0;
  for (int r0 = first; r0 < rows; r0 += ROWS) {
    if (r0 + ROWS < rows) stage(r0 + ROWS, lds[cur ^ 1]);
#pragma unroll
    for (int u = 0; u < 2; u++) {
      const int row = u * 32 + lr, R = r0 + row;
      const int pos = rows_over(min(R, rows - 1), a);
      const float2 st = a.stats[(int64_t)(tok0 + pos) * QH + kvh * a.G +
                                min(R, rows - 1) - pos * a.G];
      f32x16 s[2];
#pragma unroll
      for (int t = 0; t < 2; t++)
#pragma unroll
        for (int i = 0; i < 16; i++) s[t][i] = 0.f;
#pragma unroll
      for (int kk = 0; kk < KK; kk++) {
        const hbf16x8 qf = *reinterpret_cast<const hbf16x8*>(
            lds[cur] + row * D + flash::swz_k<D>(row, kk * 2 + h) * 8);
#pragma unroll
        for (int t = 0; t < 2; t++) s[t] = flash::mfma32(kf[t][kk], qf, s[t]);
      }
      // key wkey + 32 t + 8 (i / 4) + 4 h + i % 4 of this lane's row; the last
      // key that it sees, relative to the lane's first
      const int last = R < rows ? q_abs0 + pos - wkey - 4 * h : -1;
#pragma unroll
      for (int t = 0; t < 2; t++)
#pragma unroll
        for (int i = 0; i < 16; i++) {
          const float p =
              __builtin_amdgcn_exp2f(fmaf(s[t][i], a.c, -st.x)) * st.y;
          if (t * 32 + 8 * (i / 4) + i % 4 <= last) sum[t][i] += p;
        }
    }
    __syncthreads();
    cur ^= 1;
  }

  // ---- over the lanes' rows, then one thread per key
  float* total = reinterpret_cast<float*>(&lds[0][0]);
#pragma unroll
  for (int t = 0; t < 2; t++)
#pragma unroll
    for (int i = 0; i < 16; i++) {
      const float x = group_reduce_sum<32>(sum[t][i]);
      if (lr == 0)
        total[wave * WKEYS + t * 32 + 8 * (i / 4) + 4 * h + i % 4] = x;
    }
  __syncthreads();
  const int key = key0 + tid;
  if (key < kv_len) {
    float* w = a.key_weights +
        ((int64_t)bt[key / keys::PAGE] * a.KH + kvh) * keys::PAGE +
        key % keys::PAGE;
    *w = (key < q_abs0 ? *w : 0.f) + total[tid];
  }
}

}  // namespace

void context_attention_weights(at::Tensor out, at::Tensor q, at::Tensor k_cache,
                               at::Tensor v_cache, at::Tensor key_weights,
                               at::Tensor tile_seq, at::Tensor tile_qbase,
                               at::Tensor cu_seqlens_q, at::Tensor kv_lens,
                               at::Tensor block_tables, double scale,
                               at::Tensor sinks) {
  keys::check_weights(key_weights, block_tables);
  keys::check_pages(k_cache, v_cache, key_weights);
  keys::check_rows(out, q, k_cache, sinks);
  for (const auto& t : {tile_seq, tile_qbase, cu_seqlens_q, kv_lens})
    keys::check_int(t, q, "tiles and lengths");
  const int64_t B = block_tables.size(0), T = q.size(0), ntiles = tile_seq.numel();
  TORCH_CHECK(cu_seqlens_q.numel() == B + 1 && kv_lens.numel() == B &&
              tile_qbase.numel() == ntiles);
  flash::Args a{};
  a.QH = q.size(1);
  a.KH = k_cache.size(1);
  const int G = a.QH / a.KH, D = q.size(2);
  TORCH_CHECK(G <= 64 && T * G < (1 << 26), "rows of a step: 2^26 at most");
  if (ntiles == 0 || T == 0 || block_tables.size(1) == 0) return;
  const keys::Guard guard(q.device());
  const at::Tensor stats = at::empty({T, a.QH, 2}, q.options().dtype(at::kFloat));
  a.BS = keys::PAGE;
  a.max_blocks = block_tables.size(1);
  a.out = (short*)out.data_ptr();
  a.q = (const short*)q.data_ptr();
  a.k = k_cache.data_ptr();
  a.v = v_cache.data_ptr();
  a.q_ts = q.stride(0);
  a.q_hs = D;
  a.tile_seq = tile_seq.data_ptr<int>();
  a.tile_qbase = tile_qbase.data_ptr<int>();
  a.cu = cu_seqlens_q.data_ptr<int>();
  a.kv_lens = kv_lens.data_ptr<int>();
  a.block_tables = block_tables.data_ptr<int>();
  a.gs = flash::group_shift(a.QH, a.KH);
  a.scale = (float)scale;
  if (sinks.numel() > 0) a.sinks = sinks.data_ptr<float>();
  a.stats = (float2*)stats.data_ptr<float>();

  WeightArgs w{};
  w.q = a.q;
  w.k = a.k;
  w.key_weights = key_weights.data_ptr<float>();
  w.stats = a.stats;
  w.cu = a.cu;
  w.kv_lens = a.kv_lens;
  w.block_tables = a.block_tables;
  w.q_ts = a.q_ts;
  w.max_blocks = a.max_blocks;
  w.KH = a.KH;
  w.G = G;
  w.div_g = (unsigned)(((1ull << 32) + G - 1) / G);
  w.c = a.scale * flash::LOG2E;

  const dim3 grid(flash::grid_size(a, ntiles));
  const int64_t blocks = ((int64_t)a.max_blocks * keys::PAGE + KEYS - 1) / KEYS;
  const dim3 wgrid(blocks * a.KH, B);
  auto stream = at::hip::getCurrentHIPStream();
  auto launch = [&](auto d, auto fp8) {
    constexpr int D_ = decltype(d)::value;
    constexpr bool F_ = decltype(fp8)::value;
    constexpr int SRC = F_ ? flash::PAGED_FP8 : flash::PAGED_BF16;
    hipLaunchKernelGGL((flash::flash_prefill_kernel<D_, D_, SRC, false, false,
                            false, D_, flash::kvt<D_, D_>(), 4, true>),
                       grid, dim3(256), 0, stream, a);
    hipLaunchKernelGGL((key_weight_kernel<D_, F_>), wgrid, dim3(256), 0, stream,
                       w);
  };
  auto by_type = [&](auto d) {
    if (k_cache.dtype() == at::kByte) launch(d, std::true_type{});
    else launch(d, std::false_type{});
  };
  if (D == 64) by_type(std::integral_constant<int, 64>{});
  else if (D == 128) by_type(std::integral_constant<int, 128>{});
  else by_type(std::integral_constant<int, 256>{});
}

}  // namespace kaito

TORCH_LIBRARY_FRAGMENT(kaito, m) {
  m.def("context_attention_weights(Tensor(a!) out, Tensor q, Tensor k_cache, Tensor v_cache, Tensor(b!) key_weights, Tensor tile_seq, Tensor tile_qbase, Tensor cu_seqlens_q, Tensor kv_lens, Tensor block_tables, float scale, Tensor sinks) -> ()");
}
TORCH_LIBRARY_IMPL(kaito, CUDA, m) {
  m.impl("context_attention_weights", &kaito::context_attention_weights);
}
