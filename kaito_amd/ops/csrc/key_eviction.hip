// Cutting paged caches to a budget of keys.
//
// heavy_keys: a sequence of more than `budget` keys keeps its newest `recent` and
//   the budget - recent others with the largest weights, summed over the kv heads.
//   key_total_kernel: one thread per key sums its heads in f64 and leaves the f32
//   total as an integer of the same order. choose_keys_kernel: one workgroup per
//   sequence finds the smallest total that stays, eight bits at a time (a histogram
//   in LDS per digit), and writes the places of those above it and of as many equal
//   ones as there is room for, lowest places first, by ballots and a running count.
//   No step depends on timing.
// compact_pages: key kept[i] goes to place i, in place. `kept` ascends, so that
//   kept[i] >= i, and the sources of later places are never among earlier ones: a
//   workgroup per sequence, kv head and array takes its places tile by tile, a
//   barrier between a tile's loads and its stores, and nothing else has to wait.
#include "common.h"
#include "keys_common.h"
#include <torch/library.h>

namespace kaito {

namespace {

using keys::PAGE;

// order of f32 as unsigned integers, NaN above all
KAITO_DEV unsigned ordered(const float x) {
  if (x != x) return 0xffffffffu;
  const unsigned u = __builtin_bit_cast(unsigned, x + 0.f);   // -0 is 0
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

__global__ __launch_bounds__(256)
void key_total_kernel(unsigned* __restrict__ totals,      // [B, width * 16]
                      const float* __restrict__ key_weights,
                      const int* __restrict__ block_tables,
                      const int* __restrict__ seq_lens, const int width,
                      const int KH, const int budget) {
  const int seq = blockIdx.y, key = blockIdx.x * 256 + threadIdx.x;
  const int len = min(seq_lens[seq], width * PAGE);
  if (len <= budget || key >= len) return;
  const int page = block_tables[(int64_t)seq * width + key / PAGE];
  const float* w = key_weights + (int64_t)page * KH * PAGE + key % PAGE;
  double sum = 0.;
  for (int h = 0; h < KH; h++) sum += (double)w[h * PAGE];
  totals[(int64_t)seq * width * PAGE + key] = ordered((float)sum);
}

constexpr int CHOOSERS = 1024;

__global__ __launch_bounds__(CHOOSERS)
void choose_keys_kernel(int* __restrict__ kept, int* __restrict__ kept_lens,
                        const unsigned* __restrict__ totals,
                        const int* __restrict__ seq_lens, const int width,
                        const int budget, const int recent) {
  constexpr int WAVES = CHOOSERS / 64;
  __shared__ int hist[256];
  __shared__ int found[2];
  __shared__ int counts[2][WAVES];
  const int seq = blockIdx.x, tid = threadIdx.x;
  const int lane = tid & 63, wave = tid >> 6;
  const int len = max(0, min(seq_lens[seq], width * PAGE));
  int* out = kept + (int64_t)seq * budget;
  if (tid == 0) kept_lens[seq] = min(len, budget);
  if (len <= budget) {
    for (int i = tid; i < budget; i += CHOOSERS) out[i] = i < len ? i : -1;
    return;
  }
  const unsigned* w = totals + (int64_t)seq * width * PAGE;
  const int old = len - recent, heavy = budget - recent;  // old > heavy
  for (int i = tid; i < recent; i += CHOOSERS) out[heavy + i] = old + i;
  if (heavy == 0) return;

  // ---- `left` of those that start with `prefix` stay
  unsigned prefix = 0;
  int left = heavy;
  for (int shift = 24; shift >= 0; shift -= 8) {
    if (tid < 256) hist[tid] = 0;
    __syncthreads();
    const unsigned mask = shift == 24 ? 0u : ~0u << (shift + 8);
    for (int i = tid; i < old; i += CHOOSERS) {
      const unsigned x = w[i];
      if ((x & mask) == prefix) atomicAdd(&hist[x >> shift & 255], 1);
    }
    __syncthreads();
    if (wave == 0) {                // digits from the top, four per lane
      int n[4], mine = 0;
#pragma unroll
      for (int j = 0; j < 4; j++) mine += n[j] = hist[255 - lane * 4 - j];
      int above = mine;
#pragma unroll
      for (int off = 1; off < 64; off <<= 1) {
        const int x = __shfl_up(above, off, 64);
        if (lane >= off) above += x;
      }
      above -= mine;
#pragma unroll
      for (int j = 0; j < 4; j++) {
        if (above < left && above + n[j] >= left) {
          found[0] = 255 - lane * 4 - j;
          found[1] = left - above;
        }
        above += n[j];
      }
    }
    __syncthreads();
    prefix |= (unsigned)found[0] << shift;
    left = found[1];
    __syncthreads();
  }

  // ---- those above `prefix` and the first `left` equal ones, in order
  int at = 0, ties = 0;             // kept and equal ones before this tile
  const unsigned long long below = (1ull << lane) - 1;
  for (int base = 0; base < old; base += CHOOSERS) {
    const int i = base + tid;
    const unsigned x = i < old ? w[i] : 0u;
    const bool tie = i < old && x == prefix, more = i < old && x > prefix;
    const unsigned long long t = __ballot(tie), m = __ballot(more);
    if (lane == 0) {
      counts[0][wave] = __popcll(t);
      counts[1][wave] = __popcll(m);
    }
    __syncthreads();
    int t0 = ties, m0 = at, ts = 0, ms = 0;
    for (int v = 0; v < WAVES; v++) {
      if (v == wave) { t0 += ts; m0 += ms; }
      ts += counts[0][v];
      ms += counts[1][v];
    }
    // places before this key: those above, and the equal ones that stay
    const int tie_rank = t0 + __popcll(t & below);
    if (more || (tie && tie_rank < left))
      out[m0 + __popcll(m & below) + min(tie_rank, left)] = i;
    ties += ts;
    at += ms;
    __syncthreads();
  }
}

constexpr int MOVERS = 256;

// ROW: bytes of a key in K and V. Arrays of a (sequence, kv head): K, V, weights.
template <int ROW>
__global__ __launch_bounds__(MOVERS)
void compact_kernel(uint8_t* __restrict__ k, uint8_t* __restrict__ v,
                    float* __restrict__ key_weights,
                    const int* __restrict__ block_tables,
                    const int* __restrict__ kept,
                    const int* __restrict__ kept_lens, const int width,
                    const int places, const int pages, const int KH) {
  typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
  const int seq = blockIdx.y, kvh = blockIdx.x % KH, which = blockIdx.x / KH;
  const int n = min(kept_lens[seq], min(places, width * PAGE));
  const int* bt = block_tables + (int64_t)seq * width;
  const int* from = kept + (int64_t)seq * places;
  // a place's index among the rows of the array, < 0: none
  auto row_of = [&](const int key) -> int64_t {
    if (key < 0 || key >= width * PAGE) return -1;
    const int page = bt[key / PAGE];
    if (page < 0 || page >= pages) return -1;
    return ((int64_t)page * KH + kvh) * PAGE + key % PAGE;
  };
  auto walk = [&](auto* base, const int chunks) {
    const int step = MOVERS / chunks;
    for (int i0 = 0; i0 < n; i0 += step) {
      const int i = i0 + threadIdx.x / chunks, c = threadIdx.x % chunks;
      const int src = i < n ? from[i] : i;
      const int64_t of = src != i ? row_of(src) : -1;
      std::remove_reference_t<decltype(*base)> x{};
      if (of >= 0) x = base[of * chunks + c];
      __builtin_amdgcn_s_waitcnt(0x0f70);       // vmcnt(0): loads have arrived
      __syncthreads();
      const int64_t to = of >= 0 ? row_of(i) : -1;
      if (to >= 0) base[to * chunks + c] = x;
    }
  };
  if (which == 2) walk(key_weights, 1);
  else walk((u32x4*)(which ? v : k), ROW / 16);
}

}  // namespace

void heavy_keys(at::Tensor kept, at::Tensor kept_lens, at::Tensor key_weights,
                at::Tensor block_tables, at::Tensor seq_lens, int64_t budget,
                int64_t recent) {
  keys::check_weights(key_weights, block_tables);
  keys::check_int(seq_lens, key_weights, "seq_lens");
  keys::check_int(kept, key_weights, "kept");
  keys::check_int(kept_lens, key_weights, "kept_lens");
  const int64_t B = block_tables.size(0), width = block_tables.size(1);
  TORCH_CHECK(budget >= 1 && budget < (1ll << 30) && recent >= 0 &&
              recent <= budget, "0 <= recent <= budget, budget >= 1");
  TORCH_CHECK(seq_lens.numel() == B && kept_lens.numel() == B &&
              kept.numel() == B * budget);
  if (B == 0) return;
  const keys::Guard guard(key_weights.device());
  auto stream = at::hip::getCurrentHIPStream();
  const int64_t most = width * PAGE;
  const at::Tensor totals = at::empty({B, most}, kept.options());
  unsigned* w = (unsigned*)totals.data_ptr<int>();
  if (most > budget)
    hipLaunchKernelGGL(key_total_kernel, dim3((most + 255) / 256, B), dim3(256),
                       0, stream, w, key_weights.data_ptr<float>(),
                       block_tables.data_ptr<int>(), seq_lens.data_ptr<int>(),
                       (int)width, (int)key_weights.size(1), (int)budget);
  hipLaunchKernelGGL(choose_keys_kernel, dim3(B), dim3(CHOOSERS), 0, stream,
                     kept.data_ptr<int>(), kept_lens.data_ptr<int>(), w,
                     seq_lens.data_ptr<int>(), (int)width, (int)budget,
                     (int)recent);
}

void compact_pages(at::Tensor k_cache, at::Tensor v_cache,
                   at::Tensor key_weights, at::Tensor block_tables,
                   at::Tensor kept, at::Tensor kept_lens) {
  keys::check_weights(key_weights, block_tables);
  keys::check_pages(k_cache, v_cache, key_weights);
  keys::check_int(kept, key_weights, "kept");
  keys::check_int(kept_lens, key_weights, "kept_lens");
  const int64_t B = block_tables.size(0);
  TORCH_CHECK(kept.dim() == 2 && kept.size(0) == B && kept_lens.numel() == B);
  TORCH_CHECK(k_cache.data_ptr() != v_cache.data_ptr());
  const int64_t row = k_cache.size(3) * k_cache.element_size();
  TORCH_CHECK(row == 64 || row == 128 || row == 256 || row == 512,
              "rows of 64 to 512 bytes, a power of two");
  if (B == 0 || kept.size(1) == 0) return;
  const keys::Guard guard(key_weights.device());
  auto stream = at::hip::getCurrentHIPStream();
  const int KH = k_cache.size(1);
#define CP_ROW(R_)                                                            \
  if (row == R_)                                                              \
    hipLaunchKernelGGL((compact_kernel<R_>), dim3(3 * KH, B), dim3(MOVERS), 0, \
                       stream, (uint8_t*)k_cache.data_ptr(),                  \
                       (uint8_t*)v_cache.data_ptr(),                          \
                       key_weights.data_ptr<float>(),                         \
                       block_tables.data_ptr<int>(), kept.data_ptr<int>(),    \
                       kept_lens.data_ptr<int>(), (int)block_tables.size(1),  \
                       (int)kept.size(1), (int)k_cache.size(0), KH)
  CP_ROW(64); CP_ROW(128); CP_ROW(256); CP_ROW(512);
#undef CP_ROW
}

}  // namespace kaito

TORCH_LIBRARY_FRAGMENT(kaito, m) {
  m.def("heavy_keys(Tensor(a!) kept, Tensor(b!) kept_lens, Tensor key_weights, Tensor block_tables, Tensor seq_lens, int budget, int recent) -> ()");
  m.def("compact_pages(Tensor(a!) k_cache, Tensor(b!) v_cache, Tensor(c!) key_weights, Tensor block_tables, Tensor kept, Tensor kept_lens) -> ()");
}
TORCH_LIBRARY_IMPL(kaito, CUDA, m) {
  m.impl("heavy_keys", &kaito::heavy_keys);
  m.impl("compact_pages", &kaito::compact_pages);
}
