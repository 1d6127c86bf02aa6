// Cutting paged caches to a budget of keys.
//
// heavy_keys: a sequence of more than `budget` keys keeps its newest `recent` and
//   the budget - recent others with the largest weights, summed over the kv heads.
//   Totals, in f64 and rounded to f32, become integers of the same order
//   (key_total_kernel; for short tables the choosing launch itself). choose_keys_kernel:
//   one workgroup per sequence keeps them in registers, 2048 bins over the range of
//   totals at a time narrow down the smallest one that stays until 64 are left, which
//   one wave ranks; then the places of those above it and of as many equal ones as
//   there is room for, lowest places first, from ballots and a running sum. No step
//   depends on timing.
// compact_pages: key kept[i] goes to place i, in place. `kept` ascends, so that
//   kept[i] >= i, and the sources of later places are never among earlier ones: a
//   workgroup per sequence, kv head and array takes its places tile by tile, a
//   barrier between a tile's loads and its stores, and nothing else has to wait.
//
// What bounds them: the choice is a chain of short steps in one workgroup (load and
// sum 3.7 us, ends 1.4, a level of bins 1.3, the last few 0.3, places 1.6, the launch
// of 16 waves the rest): 10.5 us for 64 caches of 4352 keys and 8 kv heads, 23 with
// its totals for 4 of 32768, 15 for 16 of 6000 to 9000; by eight bits of the total at a
// time 15 and 71, as the totals of a cache share their leading bits and queued for a
// few bins; with all rows of registers gone through 12.7, 22 and 21. The closing
// is bound by memory where there are caches enough: 64 of 4352 keys, 8 kv heads of
// 128, 481 us, 4.5 TB/s read and written (one load of a thread under way 609); 4 of
// 700 6.2 us (20), by columns that make 512 workgroups.
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
constexpr int BINS = 2 * CHOOSERS;
constexpr int FEW = 64;             // totals whose order one wave finds

// x combined over the lanes up to this one; 0 is what changes nothing
template <typename F>
KAITO_DEV unsigned lanes_up_to(unsigned x, F f) {
#define SCAN_STEP(CTRL_, ROWS_)                                               \
  x = f(x, (unsigned)__builtin_amdgcn_update_dpp(0, (int)x, CTRL_, ROWS_, 0xf, \
                                                 false))
  SCAN_STEP(0x111, 0xf);            // row_shr 1, 2, 4, 8
  SCAN_STEP(0x112, 0xf);
  SCAN_STEP(0x114, 0xf);
  SCAN_STEP(0x118, 0xf);
  SCAN_STEP(0x142, 0xa);            // the last lane of a row to the next row
  SCAN_STEP(0x143, 0xc);            // and of the first half to the second
#undef SCAN_STEP
  return x;
}
struct Plus {
  KAITO_DEV unsigned operator()(unsigned a, unsigned b) const { return a + b; }
};
struct Larger {
  KAITO_DEV unsigned operator()(unsigned a, unsigned b) const { return max(a, b); }
};

// how many of a ballot's lanes come before this one
KAITO_DEV int lanes_below(const unsigned long long b) {
  return __builtin_amdgcn_mbcnt_hi((unsigned)(b >> 32),
                                   __builtin_amdgcn_mbcnt_lo((unsigned)b, 0));
}

// PER: keys of a thread that stay in its registers; ONE: these are all; SUMS: their
// totals are made here
template <int PER, bool ONE, bool SUMS>
__global__ __launch_bounds__(CHOOSERS)
void choose_keys_kernel(int* __restrict__ kept, int* __restrict__ kept_lens,
                        const unsigned* __restrict__ totals,
                        const float* __restrict__ key_weights,
                        const int* __restrict__ block_tables,
                        const int* __restrict__ seq_lens, const int width,
                        const int KH, const int budget, const int recent) {
  constexpr int WAVES = CHOOSERS / 64, PART = PER * CHOOSERS;
  __shared__ int hist[BINS];
  __shared__ unsigned ends[2][WAVES], few[FEW];
  __shared__ int sums[WAVES], found[3], listed;
  __shared__ int counts[2][PER * WAVES];
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

  // rows of CHOOSERS keys, by fours: those behind the last are not gone through
#define EACH_ROW(BASE_)                                                       \
  _Pragma("unroll")                                                           \
  for (int j0 = 0; j0 < PER && (BASE_) + j0 * CHOOSERS < old; j0 += 4)        \
    _Pragma("unroll") for (int j = j0; j < j0 + (PER < 4 ? PER : 4); j++)
  unsigned x[PER];                  // keys base + j * CHOOSERS + tid
  auto load = [&](const int base) {
    if constexpr (SUMS) {
      const int* bt = block_tables + (int64_t)seq * width;
      const float* at[PER];
      double sum[PER];
      EACH_ROW(base) {
        const int i = min(base + j * CHOOSERS + tid, old - 1);
        at[j] = key_weights + (int64_t)bt[i / PAGE] * KH * PAGE + i % PAGE;
        sum[j] = 0.;
      }
#pragma unroll 4
      for (int h = 0; h < KH; h++)
        EACH_ROW(base) sum[j] += (double)at[j][h * PAGE];
      EACH_ROW(base) x[j] = ordered((float)sum[j]);
    } else {
      EACH_ROW(base) {
        const int i = base + j * CHOOSERS + tid;
        x[j] = i < old ? w[i] : 0u;
      }
    }
  };
  auto parts = [&](auto each) {     // every part, read again unless it is the only one
    for (int base = 0; base < (ONE ? 1 : old); base += PART) {
      if (!ONE) load(base);
      each(base);
    }
  };
  if (ONE) load(0);

  // ---- smallest and largest total
  unsigned lo = ~0u, hi = 0u;
  parts([&](const int base) {
    EACH_ROW(base)
      if (base + j * CHOOSERS + tid < old) {
        lo = min(lo, x[j]);
        hi = max(hi, x[j]);
      }
  });
  hi = lanes_up_to(hi, Larger{});
  lo = ~lanes_up_to(~lo, Larger{});
  if (lane == 63) { ends[0][wave] = lo; ends[1][wave] = hi; }
  __syncthreads();
#pragma unroll
  for (int v = 0; v < WAVES; v++) {
    lo = v ? min(lo, ends[0][v]) : ends[0][0];
    hi = v ? max(hi, ends[1][v]) : ends[1][0];
  }

  // ---- `left` of the `some` in lo..hi stay, and all above hi
  int left = heavy, some = old;
  while (lo != hi && left != some && some > FEW) {  // uniform
    // every turn leaves 2^-11 of the range
    const int shift = max(0, 32 - __builtin_clz(hi - lo) - 11);
    *reinterpret_cast<int2*>(hist + 2 * tid) = {0, 0};
    __syncthreads();
    parts([&](const int base) {
      // A wave's equal totals would queue for one bin. Where its first row has many,
      // those of the first lane's bin are one addition.
      const int first = (x[0] - lo) >> shift;
      const bool alike = __popcll(__ballot(
          first == __builtin_amdgcn_readfirstlane(first))) > 16;
      EACH_ROW(base) {
        const unsigned d = x[j] - lo;
        if (d > hi - lo || base + j * CHOOSERS + tid >= old) continue;
        const int bin = d >> shift;
        if (!alike) {
          atomicAdd(&hist[bin], 1);
          continue;
        }
        const int one = __builtin_amdgcn_readfirstlane(bin);
        const unsigned long long same = __ballot(bin == one);
        if (bin != one) atomicAdd(&hist[bin], 1);
        else if (lanes_below(same) == 0) atomicAdd(&hist[bin], __popcll(same));
      }
    });
    __syncthreads();
    // two bins per thread, from the top
    const int2 n = *reinterpret_cast<const int2*>(hist + BINS - 2 - 2 * tid);
    int above = lanes_up_to(n.x + n.y, Plus{});
    if (lane == 63) sums[wave] = above;
    __syncthreads();
    above -= n.x + n.y;
#pragma unroll
    for (int v = 0; v < WAVES; v++) above += v < wave ? sums[v] : 0;
    const bool upper = above + n.y >= left;
    if (above < left && above + n.x + n.y >= left) {
      found[0] = BINS - 1 - 2 * tid - !upper;
      found[1] = left - above - (upper ? 0 : n.y);
      found[2] = upper ? n.y : n.x;
    }
    __syncthreads();
    lo += (unsigned)found[0] << shift;
    hi = lo + min(hi - lo, (1u << shift) - 1);      // which may end at ~0
    left = found[1];
    some = found[2];
  }
  if (lo != hi && left != some) {   // few: a wave ranks them, equal ones alike
    if (tid == 0) listed = 0;
    __syncthreads();
    parts([&](const int base) {
      EACH_ROW(base)
        if (base + j * CHOOSERS + tid < old && x[j] >= lo && x[j] <= hi)
          few[atomicAdd(&listed, 1)] = x[j];
    });
    __syncthreads();
    if (wave == 0) {
      const unsigned mine = lane < some ? few[lane] : 0u;
      int more = 0, same = 0;
#pragma unroll
      for (int o = 0; o < FEW; o++) {
        const unsigned y = __builtin_amdgcn_readlane(mine, o);
        more += o < some && y > mine;
        same += o < some && y == mine;
      }
      if (lane < some && more < left && more + same >= left) {
        found[0] = (int)mine;       // the same from every lane that holds it
        found[1] = left - more;
      }
    }
    __syncthreads();
    lo = hi = (unsigned)found[0];
    left = found[1];
  }

  // ---- those above hi and the first `left` of the others, in order
  int at = 0, ties = 0;             // kept and equal ones before this part
  __syncthreads();
  parts([&](const int base) {
    EACH_ROW(base) {
      const bool in = base + j * CHOOSERS + tid < old;
      const int t = __popcll(__ballot(in && x[j] - lo <= hi - lo));
      const int m = __popcll(__ballot(in && x[j] > hi));
      if (lane == 0) {
        counts[0][j * WAVES + wave] = t;
        counts[1][j * WAVES + wave] = m;
      }
    }
    __syncthreads();
    if (wave < 2) {                 // running sums, in the order of the keys
      int* c = counts[wave];
      int before = 0;
      const int rows = min(PER, (old - base + 4 * CHOOSERS - 1) / (4 * CHOOSERS) * 4);
      for (int k = 0; k < rows * WAVES; k += 64) {
        const int n = k + lane < rows * WAVES ? c[k + lane] : 0;
        const int sum = lanes_up_to(n, Plus{});
        if (k + lane < rows * WAVES) c[k + lane] = before + sum - n;
        before += __builtin_amdgcn_readlane(sum, 63);
      }
      if (lane == 0) found[wave] = before;
    }
    __syncthreads();
    EACH_ROW(base) {
      const int i = base + j * CHOOSERS + tid;
      const bool tie = i < old && x[j] - lo <= hi - lo;
      const bool more = i < old && x[j] > hi;
      const int rank = ties + counts[0][j * WAVES + wave] +
          lanes_below(__ballot(tie));
      const int m = at + counts[1][j * WAVES + wave] +
          lanes_below(__ballot(more));
      if (more || (tie && rank < left)) out[m + min(rank, left)] = i;
    }
    ties += found[0];
    at += found[1];
    __syncthreads();
  });
}
#undef EACH_ROW

constexpr int MOVERS = 256;
constexpr int DEEP = 8;             // loads of a thread under way at once

// Columns of K, V (CHUNKS x 16 bytes, `parts` of them make a row) or the weights
// of a (sequence, kv head).
template <int CHUNKS>
__global__ __launch_bounds__(MOVERS)
void compact_kernel(uint8_t* __restrict__ k, uint8_t* __restrict__ v,
                    float* __restrict__ key_weights,
                    const int* __restrict__ block_tables,
                    const int* __restrict__ kept,
                    const int* __restrict__ kept_lens, const int width,
                    const int places, const int pages, const int KH,
                    const int parts) {
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
  // rows of `stride` elements, of which this workgroup moves `chunks`
  auto walk = [&](auto* base, const int chunks, const int stride) {
    typedef std::remove_reference_t<decltype(*base)> T;
    const int step = MOVERS / chunks, c = threadIdx.x % chunks;
    for (int i0 = threadIdx.x / chunks; i0 - (int)threadIdx.x / chunks < n;
         i0 += step * DEEP) {
      T x[DEEP];
      int64_t of[DEEP], to[DEEP];
      int src[DEEP];
#pragma unroll
      for (int j = 0; j < DEEP; j++) {
        const int i = i0 + j * step;
        src[j] = i < n ? from[i] : i;
      }
#pragma unroll
      for (int j = 0; j < DEEP; j++) {
        const int i = i0 + j * step;
        const bool moves = i < n && src[j] != i;
        of[j] = moves ? row_of(src[j]) : -1;
        to[j] = moves ? row_of(i) : -1;
      }
#pragma unroll
      for (int j = 0; j < DEEP; j++)
        if (of[j] >= 0) x[j] = base[of[j] * stride + c];
      __builtin_amdgcn_s_waitcnt(0x0f70);       // vmcnt(0): loads have arrived
      __syncthreads();
#pragma unroll
      for (int j = 0; j < DEEP; j++)
        if (of[j] >= 0 && to[j] >= 0) base[to[j] * stride + c] = x[j];
    }
  };
  if (which == 2 * parts) {
    walk(key_weights, 1, 1);
  } else {
    const int part = which >> 1;
    walk((u32x4*)(which & 1 ? v : k) + part * CHUNKS, CHUNKS, parts * CHUNKS);
  }
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
  const int KH = key_weights.size(1);
  const float* weights = key_weights.data_ptr<float>();
  const int *tables = block_tables.data_ptr<int>(), *lens = seq_lens.data_ptr<int>();
  // as many registers as the table's keys need; short caches' totals without a
  // launch of their own
  const bool own = most <= 8 * CHOOSERS && KH <= 16;
  at::Tensor totals;
  unsigned* w = nullptr;
  if (!own && most > budget) {
    totals = at::empty({B, most}, kept.options());
    w = (unsigned*)totals.data_ptr<int>();
    hipLaunchKernelGGL(key_total_kernel, dim3((most + 255) / 256, B), dim3(256),
                       0, stream, w, weights, tables, lens, (int)width, KH,
                       (int)budget);
  }
  auto choose = [&](auto kernel) {
    hipLaunchKernelGGL(kernel, dim3(B), dim3(CHOOSERS), 0, stream,
                       kept.data_ptr<int>(), kept_lens.data_ptr<int>(), w,
                       weights, tables, lens, (int)width, KH, (int)budget,
                       (int)recent);
  };
  if (own && most <= 2 * CHOOSERS) choose(choose_keys_kernel<2, true, true>);
  else if (own) choose(choose_keys_kernel<8, true, true>);
  else if (most <= 32 * CHOOSERS) choose(choose_keys_kernel<32, true, false>);
  else choose(choose_keys_kernel<32, false, false>);
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
  const int64_t chunks = row / 16;
  // columns that a workgroup moves: as few as fill the chip, 64 bytes at least
  int64_t own = chunks;
  while (own > 4 && 2 * KH * B * (chunks / own) < 512) own /= 2;
  const int64_t parts = chunks / own;
#define CP_CHUNKS(C_)                                                         \
  if (own == C_)                                                              \
    hipLaunchKernelGGL((compact_kernel<C_>), dim3((2 * parts + 1) * KH, B),   \
                       dim3(MOVERS), 0, stream, (uint8_t*)k_cache.data_ptr(), \
                       (uint8_t*)v_cache.data_ptr(),                          \
                       key_weights.data_ptr<float>(),                         \
                       block_tables.data_ptr<int>(), kept.data_ptr<int>(),    \
                       kept_lens.data_ptr<int>(), (int)block_tables.size(1),  \
                       (int)kept.size(1), (int)k_cache.size(0), KH, (int)parts)
  CP_CHUNKS(4); CP_CHUNKS(8); CP_CHUNKS(16); CP_CHUNKS(32);
#undef CP_CHUNKS
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
