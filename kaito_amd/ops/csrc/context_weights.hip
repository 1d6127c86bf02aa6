// Attention of chunks of new tokens over the paged cache that also keeps what
// every key receives:
//   p_ij = exp(s_ij - m_i) / l_i,   o_i = sum_j p_ij v_j   (flash_prefill.h)
//   W_j (+)= sum over the rows i that see key j, all heads of a kv group, of p_ij
// A key's weights need the rows' final maximum m and sum l, so that they are a
// second pass over the scores: the first leaves (m, 1 / l) of every row.
//
// The second pass keeps the keys and lets the rows go by, so that every key's sum
// has one owner: no atomics, the same bits every time. A workgroup is 4 waves x 64
// keys (32 with 256 dims) of a kv head. S^T = K Q^T on v_mfma_f32_32x32x16_bf16:
// the wave's K stays in registers as the first operand; query rows, flattened over
// the heads of the group (row = position * G + head), come in tiles of 64 through
// LDS with their m and 1 / l, two tiles ahead (swizzled as flash_prefill.h's K). A
// lane holds one row of half a tile and 16 keys of every 32, so that m and 1 / l
// are per-lane scalars and a weight is a multiply-add, an exponential and a
// multiply-add into its key's sum.
//
// What bounds it: its products of 32 x 32 x 16. With operands of random bits one takes
// 33.6 ns on a SIMD (16.3 with constant ones): 2048 rows of 32 heads over 16384 keys
// and 8 kv heads of 128 are 261 us of them, and the pass takes 268, beside 566 of
// flash_prefill.h's twice as many. One product after another and then all weights
// 381 us; the loop without masks and addresses 315; products and weights in turns
// 298; tiles of 64 rows and fragments four products ahead of their use 268. Eight
// waves that share a tile: 278. It is not what the matrix unit can do: two products
// of 16 x 16 x 32, the same operations, take 18 ns with random operands and 25 with
// as many multiply-adds and exponentials in between. In this loop they took 287 (276
// with those gathered by fours), without copies and barriers 258, without LDS reads
// 222: there, staging and the reads of fragments are ahead of them.
//
// Weights enter the product with V as bf16, as in context_attention, and the outputs
// are its bits wherever the keys are not shared out. As value and remainder, the EXT
// form, the long chunk took 974 us for both passes instead of 785, eight of 97 to 1000
// rows 505 (423), four of 333 to 1200 over e4m3 pages and heads of 64 773 (630); the
// error against 64 bits was 1.7e-3 instead of 1.9e-3, of which the rounding of the
// output is 1.65e-3. Scores, maxima, sums and the keys' weights are f32.
#include "flash_prefill.h"
#include "keys_common.h"
#include <torch/library.h>

namespace kaito {

namespace {

using flash::hbf16x8;
using flash::f32x16;

// 32-key tiles of a wave: with 256 dims two of them do not fit the registers
template <int D> constexpr int tiles_of = D <= 128 ? 2 : 1;
constexpr int NW = 4;               // waves of a workgroup
template <int D> constexpr int keys_of = NW * 32 * tiles_of<D>;
constexpr int ROWS = 64;            // query rows of a tile, two halves

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
  float c;                          // scale * log2 e
};

// x, of which the compiler does not know that: what is made of it is made there and
// not kept in registers from ahead of the loop
KAITO_DEV int fresh(int x) {
  asm volatile("" : "+v"(x));
  return x;
}

// 32 keys per tile, those behind the last in its place: lane lr's, 8 dims in 16
template <int D, bool FP8>
KAITO_DEV void load_keys(hbf16x8 (&kf)[tiles_of<D>][D / 16], const WeightArgs& a,
                         const int* bt, const int key0, const int kv_len,
                         const int kvh, const int lr, const int h) {
#pragma unroll
  for (int t = 0; t < tiles_of<D>; t++) {
    const int key = min(key0 + t * 32 + lr, kv_len - 1);
    const int64_t row =
        ((int64_t)bt[key / keys::PAGE] * a.KH + kvh) * keys::PAGE +
        key % keys::PAGE;
#pragma unroll
    for (int kk = 0; kk < D / 16; kk++) {
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
}

// the lanes' rows together: total[key] of a wave's keys
template <int NT>
KAITO_DEV void sum_rows(float* total, const f32x16 (&sum)[NT], const int lr,
                        const int h) {
#pragma unroll
  for (int t = 0; t < NT; t++)
#pragma unroll
    for (int i = 0; i < 16; i++) {
      const float x = group_reduce_sum<32>(sum[t][i]);
      if (lr == 0) total[t * 32 + 8 * (i / 4) + 4 * h + i % 4] = x;
    }
}

KAITO_DEV void add_weight(const WeightArgs& a, const int* bt, const int kvh,
                          const int key, const int q_abs0, const float x) {
  float* w = a.key_weights +
      ((int64_t)bt[key / keys::PAGE] * a.KH + kvh) * keys::PAGE +
      key % keys::PAGE;
  *w = (key < q_abs0 ? *w : 0.f) + x;
}

// The sequence whose chunk is the n-th longest, of up to 64: workgroups of long chunks
// run longest and begin first (eight of 97 to 1000 rows, the longest last: 200 -> 171
// us; four of 333 to 1200 rows of 64/8 heads of 64, e4m3 pages: 293 -> 253).
KAITO_DEV int nth_longest(const int* cu, const int n, const int seqs) {
  if (seqs == 1 || seqs > 64) return n;
  const int lane = threadIdx.x & 63;
  const int mine = lane < seqs ? cu[lane + 1] - cu[lane] : -1;
  int before = 0;
  for (int o = 0; o < seqs; o++) {
    const int len = __builtin_amdgcn_readlane(mine, o);
    before += len > mine || (len == mine && o < lane);
  }
  return __ffsll(__ballot(lane < seqs && before == n)) - 1;
}

template <int D, bool FP8>
__global__ __launch_bounds__(NW * 64, 2)
void key_weight_kernel(const WeightArgs a) {
  constexpr int TH = NW * 64, KK = D / 16, CK = D / 8, COPIES = ROWS * CK / TH;
  constexpr int NT = tiles_of<D>, KEYS = keys_of<D>, WKEYS = KEYS / NW;
  const int seq = nth_longest(a.cu, blockIdx.y, gridDim.y);
  const int kvh = blockIdx.x % a.KH, key0 = blockIdx.x / a.KH * KEYS;
  const int tok0 = a.cu[seq], q_len = a.cu[seq + 1] - tok0;
  const int kv_len = min(a.kv_lens[seq], a.max_blocks * keys::PAGE);
  if (key0 >= kv_len || q_len <= 0) return;
  const int* bt = a.block_tables + (int64_t)seq * a.max_blocks;
  const int QH = a.KH * a.G, q_abs0 = kv_len - q_len;

  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int lr = lane & 31, h = lane >> 5;
  __shared__ __attribute__((aligned(128))) short lds[3][ROWS * D + NW * 4 * ROWS];

  // ---- this wave's keys
  const int wkey = key0 + wave * WKEYS;
  hbf16x8 kf[NT][KK];
  load_keys<D, FP8>(kf, a, bt, wkey, kv_len, kvh, lr, h);

  // ---- positions that see one of the workgroup's keys, POS of them a tile: a row's
  // position in the tile and its head do not change. Rows behind the last whole
  // position stand for it and weigh nothing.
  const int pos_n = ROWS / a.G, real = pos_n * a.G;
  const int first = max(0, key0 - q_abs0) / pos_n * pos_n;
  uint32_t q_off[COPIES];           // of this thread's copies, behind the tile's base
#pragma unroll
  for (int j = 0; j < COPIES; j++) {
    const int s = j * TH + tid, row = min(s / CK, real - 1);
    q_off[j] = (uint32_t)(row / a.G) * (uint32_t)a.q_ts + row % a.G * D +
        flash::swz_k<D>(s / CK, s % CK) * 8;
  }
  // every wave stages all pairs of (maximum, 1 / sum) for itself: a word a lane, twice
  uint32_t st_off[2];
#pragma unroll
  for (int u = 0; u < 2; u++) {
    const int row = min(u * 32 + (lane >> 1), real - 1);
    st_off[u] = (row / a.G * QH + row % a.G) * 2 + (lane & 1);
  }
  const short* q_base = a.q + (int64_t)(tok0 + first) * a.q_ts + kvh * a.G * D;
  const float* st_base = reinterpret_cast<const float*>(
      a.stats + (int64_t)(tok0 + first) * QH + kvh * a.G);
  auto copy4 = [&](const float* src, short* dst) {
    __builtin_amdgcn_global_load_lds(
        (const __attribute__((address_space(1))) unsigned int*)src,
        (__attribute__((address_space(3))) unsigned int*)dst, 4, 0, 0);
  };
  auto stage = [&](const int p0, const int b) {     // tiles in their order
    short* buf = lds[b];
    short* pairs = buf + ROWS * D + wave * 4 * ROWS;
    if (p0 + pos_n <= q_len) {
#pragma unroll
      for (int j = 0; j < COPIES; j++)
        flash::lds_copy16(q_base + q_off[j], buf + (j * TH + wave * 64) * 8);
#pragma unroll
      for (int u = 0; u < 2; u++)
        copy4(st_base + st_off[u], pairs + u * 128);
    } else if (p0 < q_len) {        // the last: behind its last position that again
      const int last = q_len - 1 - p0, me = fresh(tid);
#pragma unroll
      for (int j = 0; j < COPIES; j++) {
        const int s = j * TH + me, row = min(s / CK, real - 1);
        flash::lds_copy16(
            q_base + (int64_t)min(row / a.G, last) * a.q_ts + row % a.G * D +
                flash::swz_k<D>(s / CK, s % CK) * 8,
            buf + (j * TH + wave * 64) * 8);
      }
#pragma unroll
      for (int u = 0; u < 2; u++) {
        const int row = min(u * 32 + ((me & 63) >> 1), real - 1);
        copy4(st_base + (min(row / a.G, last) * QH + row % a.G) * 2 + (me & 1),
              pairs + u * 128);
      }
    }
    q_base += pos_n * a.q_ts;
    st_base += pos_n * QH * 2;
  };
  f32x16 sum[NT];
#pragma unroll
  for (int t = 0; t < NT; t++)
#pragma unroll
    for (int i = 0; i < 16; i++) sum[t][i] = 0.f;

  // A turn: the next half's products beside this half's weights. The matrix unit
  // works on its own once a product is issued, but two waves of a SIMD that both
  // multiply and then both weigh wait for each other (measured: the sum of both
  // times), so that every product is followed by its share of the weights: the last
  // addition of one share, the exponentials of the next, the exponents of the one
  // behind. The scheduler gathers the products otherwise. The first fragments of
  // the half after that are read on the way.
  constexpr int FEW = 4;
  hbf16x8 head[FEW];
  auto fragment = [&](const short* half, const int kk) {
    return *reinterpret_cast<const hbf16x8*>(
        half + lr * D + flash::swz_k<D>(lr, kk * 2 + h) * 8);
  };
  auto turn = [&](const short* half, const short* after, f32x16 (&next)[NT],
                  const f32x16 (&s)[NT], const float2_t st) {
    constexpr int GROUPS = NT * KK, EACH = 16 / KK;
    float x[16 * NT];
    auto exponents = [&](const int g) {
#pragma unroll
      for (int e = g * EACH; e < (g + 1) * EACH; e++)
        x[e] = fmaf(s[e / 16][e % 16], a.c, -st[0]);
    };
    auto weights = [&](const int g) {
#pragma unroll
      for (int e = g * EACH; e < (g + 1) * EACH; e++)
        sum[e / 16][e % 16] = fmaf(x[e], st[1], sum[e / 16][e % 16]);
    };
    hbf16x8 qf[KK + FEW];
#pragma unroll
    for (int kk = 0; kk < FEW; kk++) qf[kk] = head[kk];
    exponents(0);
#pragma unroll
    for (int t = 0; t < NT; t++)
#pragma unroll
      for (int i = 0; i < 16; i++) next[t][i] = 0.f;
#pragma unroll
    for (int g = 0; g < GROUPS; g++) {
      __builtin_amdgcn_sched_barrier(0);
      const int kk = g / NT, t = g % NT;
      if (t == 0)
        qf[kk + FEW] = kk + FEW < KK ? fragment(half, kk + FEW)
                                     : fragment(after, kk + FEW - KK);
      next[t] = flash::mfma32(kf[t][kk], qf[kk], next[t]);
      if (g > 0) weights(g - 1);
#pragma unroll
      for (int e = g * EACH; e < (g + 1) * EACH; e++)
        x[e] = __builtin_amdgcn_exp2f(x[e]);
      if (g + 1 < GROUPS) exponents(g + 1);
    }
    weights(GROUPS - 1);
#pragma unroll
    for (int kk = 0; kk < FEW; kk++) head[kk] = qf[KK + kk];
  };

  // In the step of a tile the next one is there and the one after it under way.
  int at = 0, p0 = first;           // place of the tile at p0 among the three
  stage(p0, 0);
  stage(p0 + pos_n, 1);
  __syncthreads();
  auto pair = [&](const short* tile, const int row) {
    float2_t st = __builtin_bit_cast(
        float2_t, *reinterpret_cast<const short4_t*>(
                      tile + ROWS * D + wave * 4 * ROWS + 4 * row));
    if (row >= real) st[1] = 0.f;
    return st;
  };
  auto ahead = [&] { stage(p0 + 2 * pos_n, at == 0 ? 2 : at - 1); };
  auto onward = [&] {
    __syncthreads();
    at = at == 2 ? 0 : at + 1;
    p0 += pos_n;
  };
  auto clear = [&](f32x16 (&s)[NT]) {
#pragma unroll
    for (int t = 0; t < NT; t++)
#pragma unroll
      for (int i = 0; i < 16; i++) s[t][i] = 0.f;
  };
  // A tile whose rows do not all see all of the wave's keys: scores are of key
  // wkey + 32 t + 8 (i / 4) + 4 h + i % 4, rows see those up to their position.
  auto edge = [&] {
    ahead();
    for (int u = 0; u < 2; u++) {
      const int row = u * 32 + lr;
      const float2_t st = pair(lds[at], row);
      f32x16 s[NT];
      clear(s);
#pragma unroll
      for (int kk = 0; kk < KK; kk++)
#pragma unroll
        for (int t = 0; t < NT; t++)
          s[t] = flash::mfma32(kf[t][kk], fragment(lds[at] + u * 32 * D, kk),
                               s[t]);
      const int pos = p0 + min(row, real - 1) / a.G;
      const int last = pos < q_len ? q_abs0 + pos - wkey - 4 * h : -1;
#pragma unroll
      for (int t = 0; t < NT; t++)
#pragma unroll
        for (int i = 0; i < 16; i++) {
          float x = fmaf(s[t][i], a.c, -st[0]);
          if (t * 32 + 8 * (i / 4) + i % 4 > last) x = -INFINITY;
          sum[t][i] = fmaf(__builtin_amdgcn_exp2f(x), st[1], sum[t][i]);
        }
    }
    onward();
  };
  while (p0 < q_len && q_abs0 + p0 < key0 + KEYS - 1) edge();
  if (p0 + pos_n <= q_len) {
    f32x16 s0[NT], s1[NT];
    clear(s0);
#pragma unroll
    for (int kk = 0; kk < KK; kk++)
#pragma unroll
      for (int t = 0; t < NT; t++)
        s0[t] = flash::mfma32(kf[t][kk], fragment(lds[at], kk), s0[t]);
#pragma unroll
    for (int kk = 0; kk < FEW; kk++) head[kk] = fragment(lds[at] + 32 * D, kk);
    do {
      const short *tile = lds[at], *next = lds[at == 2 ? 0 : at + 1];
      const float2_t st0 = pair(tile, lr), st1 = pair(tile, 32 + lr);
      ahead();
      turn(tile + 32 * D, next, s1, s0, st0);
      turn(next, next + 32 * D, s0, s1, st1);
      onward();
    } while (p0 + pos_n <= q_len);
  }
  if (p0 < q_len) edge();
  __syncthreads();

  // ---- over the lanes' rows, then one thread per key
  float* total = reinterpret_cast<float*>(&lds[0][0]);
  sum_rows<NT>(total + wave * WKEYS, sum, lr, h);
  __syncthreads();
  const int key = key0 + tid;
  if (tid < KEYS && key < kv_len) add_weight(a, bt, kvh, key, q_abs0, total[tid]);
}

// The same for steps that the kernel above leaves most of the chip without work in:
// 8 waves share 64 keys and take 32 rows each in turn, straight from memory and a
// turn ahead; their sums meet in LDS. No tile waits for another wave.
template <int D, bool FP8>
__global__ __launch_bounds__(512, 2)
void key_weight_few_kernel(const WeightArgs a) {
  constexpr int KK = D / 16, NT = tiles_of<D>, WKEYS = 32 * NT;
  const int seq = blockIdx.y;
  const int kvh = blockIdx.x % a.KH, key0 = blockIdx.x / a.KH * WKEYS;
  const int tok0 = a.cu[seq], q_len = a.cu[seq + 1] - tok0;
  const int kv_len = min(a.kv_lens[seq], a.max_blocks * keys::PAGE);
  if (key0 >= kv_len || q_len <= 0) return;
  const int* bt = a.block_tables + (int64_t)seq * a.max_blocks;
  const int QH = a.KH * a.G, q_abs0 = kv_len - q_len;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int lr = lane & 31, h = lane >> 5;
  __shared__ float total[8][WKEYS];

  const int rows = q_len * a.G, first = max(0, key0 - q_abs0) * a.G + wave * 32;
  hbf16x8 qf[KK];
  float2 st = {0.f, 0.f};
  int last = -1;
  auto fetch = [&](const int r0) {  // this lane's row, the last one in its place
    const int R = r0 + lr, in = min(R, rows - 1);
    const int pos = in / a.G, head = kvh * a.G + in % a.G;
    const short* p = a.q + (int64_t)(tok0 + pos) * a.q_ts + head * D + h * 8;
#pragma unroll
    for (int kk = 0; kk < KK; kk++)
      qf[kk] = *reinterpret_cast<const hbf16x8*>(p + kk * 16);
    st = a.stats[(int64_t)(tok0 + pos) * QH + head];
    last = R < rows ? q_abs0 + pos - key0 - 4 * h : -1;
  };
  fetch(first);
  hbf16x8 kf[NT][KK];
  load_keys<D, FP8>(kf, a, bt, key0, kv_len, kvh, lr, h);

  f32x16 sum[NT];
#pragma unroll
  for (int t = 0; t < NT; t++)
#pragma unroll
    for (int i = 0; i < 16; i++) sum[t][i] = 0.f;
  for (int r0 = first; r0 < rows; r0 += 8 * 32) {
    f32x16 s[NT];
#pragma unroll
    for (int t = 0; t < NT; t++)
#pragma unroll
      for (int i = 0; i < 16; i++) s[t][i] = 0.f;
#pragma unroll
    for (int kk = 0; kk < KK; kk++)
#pragma unroll
      for (int t = 0; t < NT; t++)
        s[t] = flash::mfma32(kf[t][kk], qf[kk], s[t]);
    const float2 now = st;
    const int seen = last;
    if (r0 + 8 * 32 < rows) fetch(r0 + 8 * 32);
#pragma unroll
    for (int t = 0; t < NT; t++)
#pragma unroll
      for (int i = 0; i < 16; i++) {
        float x = fmaf(s[t][i], a.c, -now.x);
        if (t * 32 + 8 * (i / 4) + i % 4 > seen) x = -INFINITY;
        sum[t][i] = fmaf(__builtin_amdgcn_exp2f(x), now.y, sum[t][i]);
      }
  }
  sum_rows<NT>(total[wave], sum, lr, h);
  __syncthreads();
  const int key = key0 + tid;
  if (tid < WKEYS && key < kv_len) {
    float all = 0.f;
#pragma unroll
    for (int w = 0; w < 8; w++) all += total[w][tid];
    add_weight(a, bt, kvh, key, q_abs0, all);
  }
}

// The shares' outputs of a row and head joined, and what makes weights of its
// scores. WPR waves a row: many shares are read in as few waits as four waves need.
// Lane s has share s's maximum and sum.
template <int D, int WPR>
__global__ __launch_bounds__(256)
void join_kernel(short* __restrict__ out, float2* __restrict__ stats,
                 const float2* __restrict__ parts, const float* __restrict__ part,
                 const int* __restrict__ ends, const int QH, const int splits,
                 const int64_t rows) {
  constexpr int EACH = D / 64;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t row = WPR == 1 ? (int64_t)blockIdx.x * 4 + wave : blockIdx.x;
  __shared__ float sums[WPR == 1 ? 1 : WPR][D];
  if (row >= (int64_t)*ends * QH) return;       // behind the last sequence: not ours
  const float2 mine = parts[min(lane, splits - 1) * rows + row];
  const float m = wave_reduce_max(mine.x);
  // a share whose sum is 0 has left no output; one that is no number counts, however
  // small its maximum
  const float e = lane >= splits || mine.y == 0.f ? 0.f
      : mine.y == mine.y ? __builtin_amdgcn_exp2f(mine.x - m) : mine.y;
  const float sum = wave_reduce_sum(e == 0.f ? 0.f : e * mine.y);
  const float inv = 1.f / fmaxf(sum, 1e-30f);
  float o[EACH];
#pragma unroll
  for (int i = 0; i < EACH; i++) o[i] = 0.f;
#pragma unroll 8
  for (int s = WPR == 1 ? 0 : wave; s < splits; s += WPR) {
    const float w = __builtin_bit_cast(
        float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, e), s));
    const float* p = part + (s * rows + row) * D + lane * EACH;
#pragma unroll
    for (int i = 0; i < EACH; i++) o[i] = fmaf(w, w == 0.f ? 0.f : p[i], o[i]);
  }
  if constexpr (WPR > 1) {
#pragma unroll
    for (int i = 0; i < EACH; i++) sums[wave][lane * EACH + i] = o[i];
    __syncthreads();
    if (wave > 0) return;
#pragma unroll
    for (int i = 0; i < EACH; i++)
#pragma unroll
      for (int v = 1; v < WPR; v++) o[i] += sums[v][lane * EACH + i];
  }
#pragma unroll
  for (int i = 0; i < EACH; i++)
    out[row * D + lane * EACH + i] = f32_to_bf16(o[i] * inv);
  if (lane == 0) stats[row] = {sum == sum ? m : sum, inv};
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
  TORCH_CHECK(G <= ROWS, "unsupported GQA group ", G);
  TORCH_CHECK(T < (1ll << 31), "q: too many rows");
  TORCH_CHECK(q.stride(0) < (1 << 25), "q: rows 2^25 apart at most");
  if (ntiles == 0 || T == 0) return;
  const keys::Guard guard(q.device());
  if (block_tables.size(1) == 0) {  // no row has a key
    out.zero_();
    return;
  }
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
  w.c = a.scale * flash::LOG2E;

  // Few workgroups share out the keys too: as many shares as make two workgroups of
  // a CU, of four tiles of the table's keys at least.
  const int64_t groups = flash::grid_size(a, ntiles);
  const int64_t tiles = (int64_t)a.max_blocks * keys::PAGE / (D <= 128 ? 64 : 32);
  a.splits = std::max<int64_t>(
      1, std::min<int64_t>({512 / groups, tiles / 4, 64}));
  a.rows = (int)T;
  at::Tensor part, parts;
  if (a.splits > 1) {
    const auto f32 = q.options().dtype(at::kFloat);
    part = at::empty({a.splits, T, a.QH, D}, f32);
    parts = at::empty({a.splits, T, a.QH, 2}, f32);
    a.part = part.data_ptr<float>();
    a.stats = (float2*)parts.data_ptr<float>();
  }
  const dim3 grid(groups, a.splits);
  auto stream = at::hip::getCurrentHIPStream();
  auto launch = [&](auto d, auto fp8) {
    constexpr int D_ = decltype(d)::value;
    constexpr bool F_ = decltype(fp8)::value;
    constexpr int SRC = F_ ? flash::PAGED_FP8 : flash::PAGED_BF16;
    hipLaunchKernelGGL((flash::flash_prefill_kernel<D_, D_, SRC, false, false,
                            false, D_, flash::kvt<D_, D_>(), 4, true>),
                       grid, dim3(256), 0, stream, a);
    const int64_t rows = T * a.QH;
    auto join = [&](auto kernel, const int64_t groups) {
      hipLaunchKernelGGL(kernel, dim3(groups), dim3(256), 0, stream, a.out,
                         (float2*)stats.data_ptr<float>(), a.stats, a.part,
                         a.cu + B, a.QH, a.splits, rows);
    };
    if (a.splits > 8) join(join_kernel<D_, 4>, rows);
    else if (a.splits > 1) join(join_kernel<D_, 1>, (rows + 3) / 4);
    constexpr int KEYS = keys_of<D_>, SHARED = 32 * tiles_of<D_>;
    const int64_t held = (int64_t)a.max_blocks * keys::PAGE;
    auto blocks = [&](const int keys) {
      return dim3((held + keys - 1) / keys * a.KH, B);
    };
    // Both passes in us, by 256 keys a workgroup (128 with 256 dims) and by shared 64
    // (32), at 64 and 128 workgroups of the former. 32/8 heads of 128, 128 rows 46.0
    // and 40.7, 58.5 and 64.8, 1024 rows 136 and 105, 170 and 174; 28/4 of 128, 1024
    // rows 248 and 188, 362 and 358; 32/32 of 64, 128 rows 32.5 and 28.7, 33.1 and
    // 34.8; 8/4 of 256, 1024 rows 120 and 117, 151 and 182. At 192 shared ones lose by
    // up to 37 %, but for groups of 8 heads of 64, which would rather share up to
    // there: 1024 rows 161 and 93, 202 and 169, at 192 243 and 242. The table's width
    // stands for the lengths, which are on the device: where sequences are much
    // shorter, workgroups of the first kind are left without keys.
    if (blocks(KEYS).x * B < 96)
      hipLaunchKernelGGL((key_weight_few_kernel<D_, F_>), blocks(SHARED),
                         dim3(512), 0, stream, w);
    else
      hipLaunchKernelGGL((key_weight_kernel<D_, F_>), blocks(KEYS), dim3(NW * 64),
                         0, stream, w);
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
