// Products of 8-bit integers with scales: out[i][j] = (sum over k of a[i][k] w[j][k]) a_scale[i] w_scale[j], sums exact in
// 32-bit integers, scaled in float32 and rounded once to the result's type.
#include <cuda_bf16.h>

#include "blackwell.cuh"

namespace rlenv {
namespace {

struct Int8Product {
  int64_t m, k, f;
  const int8_t *a, *w;
  int64_t a_pitch, w_pitch;
  const float *a_scale, *w_scale;
  void* out;
};

// Bytes c .. c + 15 of a row of k, zeros past its end.
RLENV_D int4 sixteen(const int8_t* row, int64_t c, int64_t k) {
  if (c + 16 <= k) return __ldg(reinterpret_cast<const int4*>(row + c));
  int w[4] = {0, 0, 0, 0};
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (c + 4 * i + 4 <= k) w[i] = __ldg(reinterpret_cast<const int*>(row + c) + i);
  const int64_t rest = k & ~int64_t(3);  // the last word's one to three bytes
  int last = 0;
#pragma unroll
  for (int i = 0; i < 3; ++i)
    if (rest >= c && rest + i < k) last |= (int(row[rest + i]) & 0xff) << 8 * i;
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (c + 4 * i == rest) w[i] = last;
  return make_int4(w[0], w[1], w[2], w[3]);
}
RLENV_D int dot(int4 a, int4 b, int sum) {
  return __dp4a(a.w, b.w, __dp4a(a.z, b.z, __dp4a(a.y, b.y, __dp4a(a.x, b.x, sum))));
}
RLENV_D void put(float* to, float x) { *to = x; }
RLENV_D void put(__nv_bfloat16* to, float x) { *to = __float2bfloat16_rn(x); }

// Few rows: a warp for kChannels channels, which reads their weights once for kRows rows; kAhead of its steps of 512 bytes are
// on their way together. One row is bound by reading the weights: 8,192 x 8,192 14.9 us (4.5 TB/s; four channels a warp 17.0,
// a channel 18.5, four steps ahead 20.2), 4,096 x 4,096 4.4, 1,024 x 4,096 from L2 2.3. More rows by their dot products.
template <typename T, int kRows, int kChannels, int kAhead>
__global__ void __launch_bounds__(128) few_rows_kernel(const __grid_constant__ Int8Product p) {
  const int lane = threadIdx.x % 32;
  const int64_t f0 = (int64_t(blockIdx.x) * 4 + threadIdx.x / 32) * kChannels;
  if (f0 >= p.f) return;
  int sums[kRows][kChannels] = {};
  for (int64_t c0 = 16 * lane; c0 < p.k; c0 += 512 * kAhead) {
    int4 w[kAhead][kChannels];
#pragma unroll
    for (int u = 0; u < kAhead; ++u)
#pragma unroll
      for (int j = 0; j < kChannels; ++j) {
        const int64_t c = c0 + 512 * u;
        w[u][j] = f0 + j < p.f && c < p.k ? sixteen(p.w + (f0 + j) * p.w_pitch, c, p.k) : make_int4(0, 0, 0, 0);
      }
#pragma unroll
    for (int u = 0; u < kAhead; ++u)
#pragma unroll
      for (int i = 0; i < kRows; ++i) {
        const int64_t c = c0 + 512 * u;
        if (i >= p.m || c >= p.k) break;
        const int4 a = sixteen(p.a + i * p.a_pitch, c, p.k);
#pragma unroll
        for (int j = 0; j < kChannels; ++j) sums[i][j] = dot(a, w[u][j], sums[i][j]);
      }
  }
#pragma unroll
  for (int i = 0; i < kRows; ++i)
#pragma unroll
    for (int j = 0; j < kChannels; ++j) {
      const int sum = __reduce_add_sync(0xffffffffu, sums[i][j]);
      if (lane == 0 && i < p.m && f0 + j < p.f)
        put(static_cast<T*>(p.out) + i * p.f + f0 + j, float(sum) * p.a_scale[i] * p.w_scale[f0 + j]);
    }
}

// ---- many rows: tensor cores ---------------------------------------------------------------------------
//
// Pairs of SMs (tcgen05, cta_group::2) multiply tiles of 256 channels by kTokens tokens, 128 terms a step: a tensor copy's
// row of 128 bytes is a step of a row. Two forms:
// - channels are the accumulator's lanes and tokens its columns: a warp's lanes hold neighbouring channels of a token and
//   store them as they are, wherever a row of the result starts. Tiles of few tokens are possible.
// - kWide: tokens are its lanes, 256 of them, and channels its columns: a lane holds neighbouring channels of its token,
//   and a warp's 32 rows of 128 bytes go out through shared memory as one tensor copy. For rows of the result on 16-byte
//   boundaries. An element costs 3 instructions instead of 7 (8,192 x 256 x 4,096 bf16, all epilogue: 35 us with the other).

constexpr int kChannelsEach = 128, kStepBytes = 128;  // of a tile, in each block of a pair
template <int kTokens, bool kWide>
struct Int8Tile {
  static_assert(!kWide || kTokens == 256, "wide tiles are 256 x 256");
  static constexpr int kHalf = kTokens / 2;  // rows of the second operand that each block copies
  static constexpr int kABytes = kChannelsEach * kStepBytes, kRingBytes = kABytes + kHalf * kStepBytes;
  static constexpr int kStages = kWide ? 5 : 6 * 32768 / kRingBytes < 10 ? 6 * 32768 / kRingBytes : 10;
  static constexpr int kEpilogue = kTokens >= 128 ? 16 : kTokens >= 64 ? 8 : 4;  // warps
  static constexpr int kMine = kTokens / (kEpilogue / 4);         // columns of a thread
  static constexpr int kThreads = 128 + 32 * kEpilogue;
  static constexpr int kColumns = 2 * kTokens;                    // two accumulators
  static constexpr int kStageBytes = kWide ? 32 * 128 : 0;        // of a warp, for its rows' way out
  // the ring starts on a 1,024-byte boundary
  static constexpr int kSmem = kStages * kRingBytes + kEpilogue * kStageBytes + 1024;
};

struct alignas(64) Int8Tiles {
  CUtensorMap a, w, result;  // result: wide tiles only
  int64_t m, f;
  const float *a_scale, *w_scale;
  void* out;
  int* parts;  // (splits, M, F) where splits > 1
  int token_tiles, channel_tiles, splits, steps, split_steps;
};

// Stands in the parts' sums for one that a wait that ran out has lost: no sum of 131,071 products reaches it.
constexpr int kLost = int(0x80000000u);

// A tile's place: taken in bands of kBand tiles of tokens, channels by channels, so that those in flight share operands
// that lie in L2.
constexpr int kBand = 8;
struct Int8Work {
  int token, channel, split, k0, steps;
  RLENV_D Int8Work(const Int8Tiles& p, int item) {
    const int tiles = p.token_tiles * p.channel_tiles;
    split = item / tiles, item %= tiles;
    const int per = kBand * p.channel_tiles, band = item / per, in = item % per, high = min(kBand, p.token_tiles - band * kBand);
    token = band * kBand + in % high, channel = in / high;
    k0 = split * p.split_steps, steps = min(p.split_steps, p.steps - k0);
  }
};

template <typename T, int kTokens, bool kWide>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(Int8Tile<kTokens, kWide>::kThreads, 1)
tile_kernel(const __grid_constant__ Int8Tiles p, int items) {
  using C = Int8Tile<kTokens, kWide>;
  extern __shared__ unsigned char raw[];
  __shared__ __align__(8) uint64_t bars[2 * C::kStages + 5];
  __shared__ uint32_t tmem_slot;
  __shared__ int dead_flag;
  __shared__ bw::Ending endings[2];  // of the pair's first block, and of its second
  __shared__ __align__(16) float scales[kWide ? 4 : C::kEpilogue][kWide ? 64 : 32];  // of a part's channels; of a run's tokens
  volatile int* const dead = &dead_flag;
  const uint32_t ring = (bw::shared_at(raw) + 1023) & ~1023u;
  const uint32_t full = bw::shared_at(bars), empty = full + 8 * C::kStages;
  const uint32_t summed = empty + 8 * C::kStages, taken = summed + 16, drained = taken + 16;
  const int warp = __shfl_sync(0xffffffffu, int(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;
  const int rank = int(bw::cluster_rank()), pairs = gridDim.x / 2;
  if (threadIdx.x == 0) {
    for (int i = 0; i < C::kStages; ++i) bw::barrier_init(full + 8 * i, 1), bw::barrier_init(empty + 8 * i, 1);
    for (int i = 0; i < 2; ++i) bw::barrier_init(summed + 8 * i, 1), bw::barrier_init(taken + 8 * i, 2 * C::kEpilogue);
    bw::barrier_init(drained, 1);
    dead_flag = 0, endings[rank] = bw::Ending{};
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 2) bw::tmem_alloc<C::kColumns>(bw::shared_at(&tmem_slot));
  bw::fence_before();
  __syncthreads();
  bw::cluster_sync();
  bw::fence_after();
  const uint32_t tmem = __shfl_sync(0xffffffffu, tmem_slot, 0);

  if (warp == 0) {
    // Both blocks copy their half of the lanes' rows and of the columns'; all bytes count at the first block's barrier.
    int stage = 0, filled = 0;
    uint32_t phase = 0;
    bool ok = true;
    const uint32_t full_at = bw::in_block(full, 0);
    for (int item = blockIdx.x / 2; item < items && ok; item += pairs) {
      const Int8Work w(p, item);
      const CUtensorMap *const lanes = kWide ? &p.a : &p.w, *const columns = kWide ? &p.w : &p.a;
      const int lane0 = (2 * (kWide ? w.token : w.channel) + rank) * kChannelsEach,
                column0 = (kWide ? w.channel : w.token) * kTokens + rank * C::kHalf;
      for (int it = 0; it < w.steps; ++it) {
        const int k = (w.k0 + it) * kStepBytes;
        const uint32_t bar = full_at + 8 * stage, a = ring + stage * C::kRingBytes;
        if (!(ok = bw::barrier_wait_warp(empty + 8 * stage, phase ^ 1, dead))) break;
        if (bw::elect()) {
          if (rank == 0) bw::barrier_expect(full + 8 * stage, 2 * C::kRingBytes);
          bw::copy_tile(a, lanes, bar, k, lane0, 0);
          bw::copy_tile(a + C::kABytes, columns, bar, k, column0, 0);
        }
        ++filled;
        if (++stage == C::kStages) stage = 0, phase ^= 1;
      }
    }
    // Each block waits for the last release of every buffer: no arrival is on its way to a block that has ended.
    for (int i = 0; i < C::kStages && ok; ++i)
      if (i < filled) ok = bw::barrier_wait_warp(empty + 8 * i, i < stage ? phase : phase ^ 1, dead);
    if (lane == 0) endings[rank].filled = filled;
  } else if (warp == 1) {
    if (rank == 0) {
      int stage = 0, buffer = 0, released = 0, runs = 0;
      uint32_t phase = 0, buffer_phase = 0;
      bool ok = true;
      constexpr uint32_t kind = bw::product_kind_int8(2 * kChannelsEach, kTokens);
      const uint32_t a0 = bw::operand(ring, false, 0), b0 = bw::operand(ring + C::kABytes, false, 0);
      for (int item = blockIdx.x / 2; item < items && ok; item += pairs) {
        const Int8Work w(p, item);
        if (!(ok = bw::barrier_wait_warp(taken + 8 * buffer, buffer_phase ^ 1, dead))) break;
        const uint32_t d = tmem + buffer * kTokens;
        for (int it = 0; it < w.steps; ++it) {
          if (!(ok = bw::barrier_wait_warp(full + 8 * stage, phase, dead))) break;
          bw::fence_after();
          const uint32_t a = a0 + stage * (C::kRingBytes / 16), b = b0 + stage * (C::kRingBytes / 16);
          const bool first = it == 0, last = it == w.steps - 1;
          if (bw::elect()) {
#pragma unroll
            for (int k = 0; k < kStepBytes / 32; ++k) bw::multiply_int8(d, a + 2 * k, b + 2 * k, kind, k > 0 || !first);
            bw::commit(empty + 8 * stage);
            if (last) bw::commit(summed + 8 * buffer);
          }
          ++released, runs += last;
          if (++stage == C::kStages) stage = 0, phase ^= 1;
        }
        if (++buffer == 2) buffer = 0, buffer_phase ^= 1;
      }
      if (lane == 0) endings[0].released = released, endings[0].runs = runs;
    }
  } else if (warp >= 4) {
    const int quarter = warp & 3, part = (warp - 4) >> 2;
    float* const own_scales = scales[kWide ? part : warp - 4];
    unsigned char* const own_stage = raw + (ring - bw::shared_at(raw)) + C::kStages * C::kRingBytes + (warp - 4) * C::kStageBytes;
    int buffer = 0;
    uint32_t buffer_phase = 0;
    bool ok = true;
    const uint32_t taken_at = bw::in_block(taken, 0), lanes = uint32_t(32 * quarter) << 16;
    for (int item = blockIdx.x / 2; item < items; item += pairs) {
      const Int8Work w(p, item);
      if constexpr (kWide) {
        constexpr int kValues = 128 / int(sizeof(T));  // of a row in a copy
        const int64_t token = int64_t(2 * w.token + rank) * kChannelsEach + 32 * quarter;
        const int64_t channel0 = int64_t(w.channel) * kTokens + part * C::kMine;
        float a_scale = token + lane < p.m ? __ldg(p.a_scale + token + lane) : 0.0f;
        // The part's four warps have its channels' scales in common.
        const auto part_sync = [&] { asm volatile("bar.sync %0, 128;" ::"r"(1 + part) : "memory"); };
        part_sync();  // the last tile's are read
        if (quarter < C::kMine / 32)
          own_scales[32 * quarter + lane] = channel0 + 32 * quarter + lane < p.f ? __ldg(p.w_scale + channel0 + 32 * quarter + lane) : 0.0f;
        ok = ok && bw::barrier_wait_warp(summed + 8 * buffer, buffer_phase, dead);
        if (!ok) a_scale = __uint_as_float(0x7fffffffu);
        bw::fence_after();
        part_sync();
        const uint64_t of_row = pair_of(a_scale, a_scale);
#pragma unroll
        for (int run = 0; run < C::kMine / 32; ++run) {
          const uint32_t at = tmem + lanes + buffer * kTokens + part * C::kMine + 32 * run;
          uint32_t v[32];
          bw::tmem_load16x2(v, at, at + 16);
          bw::tmem_ready(v);
          if (32 * run % kValues == 0) bw::store_wait_read();  // the last copy has read its rows
          __syncwarp();
#pragma unroll
          for (int i = 0; i < 32; i += 16 / int(sizeof(T))) {  // 16 bytes of a row
            uint32_t out[4];
#pragma unroll
            for (int j = 0; j < 16 / int(sizeof(T)); j += 2) {
              const float2 s = *reinterpret_cast<const float2*>(own_scales + 32 * run + i + j);
              const float2 x = values_of(multiply_pairs(
                  multiply_pairs(pair_of(float(int(v[i + j])), float(int(v[i + j + 1]))), of_row), pair_of(s.x, s.y)));
              if constexpr (sizeof(T) == 4) {
                out[j] = __float_as_uint(x.x), out[j + 1] = __float_as_uint(x.y);
              } else {
                const __nv_bfloat162 pair = __floats2bfloat162_rn(x.x, x.y);
                out[j / 2] = *reinterpret_cast<const uint32_t*>(&pair);
              }
            }
            // 16-byte pieces of a row are exchanged by the row's low three bits, as the copy takes them
            const int piece = (32 * run % kValues + i) * int(sizeof(T)) / 16;
            *reinterpret_cast<uint4*>(own_stage + lane * 128 + ((piece ^ (lane & 7)) << 4)) = make_uint4(out[0], out[1], out[2], out[3]);
          }
          if ((32 * run + 32) % kValues == 0) {
            bw::fence_async();
            __syncwarp();
            const int64_t channel = channel0 + 32 * run + 32 - kValues;
            if (lane == 0 && token < p.m && channel < p.f) bw::store_tile(&p.result, bw::shared_at(own_stage), int(channel), int(token));
            bw::store_commit();
          }
        }
      } else {
        const int64_t channel = int64_t(2 * w.channel + rank) * kChannelsEach + 32 * quarter + lane;
        const bool there = channel < p.f;
        const float w_scale = there && p.splits == 1 ? __ldg(p.w_scale + channel) : 0.0f;
        ok = ok && bw::barrier_wait_warp(summed + 8 * buffer, buffer_phase, dead);
        bw::fence_after();
#pragma unroll
        for (int run = 0; run < C::kMine / 32; ++run) {
          const int column = part * C::kMine + 32 * run;
          const int64_t t0 = int64_t(w.token) * kTokens + column;
          const int count = int(min(int64_t(32), p.m - t0));
          if (count <= 0) break;
          uint32_t v[32];
          const uint32_t at = tmem + lanes + buffer * kTokens + column;
          bw::tmem_load16x2(v, at, at + 16);
          __syncwarp();
          own_scales[lane] = !ok ? __uint_as_float(0x7fffffffu) : lane < count ? __ldg(p.a_scale + t0 + lane) : 0.0f;
          __syncwarp();
          bw::tmem_ready(v);
          if (p.splits == 1) {
            T* const to = static_cast<T*>(p.out) + t0 * p.f + channel;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              const float4 s = reinterpret_cast<const float4*>(own_scales)[i];
              const float of[4] = {s.x, s.y, s.z, s.w};
#pragma unroll
              for (int j = 0; j < 4; ++j)
                if (there && 4 * i + j < count) put(to + (4 * i + j) * p.f, float(int(v[4 * i + j])) * of[j] * w_scale);
            }
          } else {
            int* const to = p.parts + (int64_t(w.split) * p.m + t0) * p.f + channel;
#pragma unroll
            for (int i = 0; i < 32; ++i)
              if (there && i < count) to[i * p.f] = ok ? int(v[i]) : kLost;
          }
          __syncwarp();
        }
      }
      bw::fence_before();
      __syncwarp();
      if (ok && lane == 0) bw::barrier_arrive(taken_at + 8 * buffer);
      if (++buffer == 2) buffer = 0, buffer_phase ^= 1;
    }
    if constexpr (kWide) bw::store_wait();
  }
  __syncwarp();
  bw::fence_before();
  __syncthreads();
  if (threadIdx.x == 0) {
    endings[rank].gave_up = dead_flag;
    if (dead_flag) bw::note_given_up();
    bw::tell(&endings[rank], rank ^ 1);
  }
  bw::cluster_sync();
  bw::fence_after();
  if (endings[0].gave_up || endings[1].gave_up)
    bw::drain<C::kStages>(endings, rank, warp, full, C::kRingBytes, empty, summed, drained);
  if (warp == 2) bw::tmem_free<C::kColumns>(tmem);
}

// The result from the parts' sums.
template <typename T>
__global__ void __launch_bounds__(256) add_parts_kernel(const int* __restrict__ parts, int splits, int64_t m, int64_t f,
                                                        const float* __restrict__ a_scale, const float* __restrict__ w_scale,
                                                        T* __restrict__ out) {
  const int64_t e = int64_t(blockIdx.x) * 256 + threadIdx.x;
  if (e >= m * f) return;
  int sum = 0;
  bool lost = false;
#pragma unroll 8
  for (int s = 0; s < splits; ++s) {
    const int part = __ldg(parts + s * m * f + e);
    sum += part, lost |= part == kLost;
  }
  const int64_t t = e / f;
  const float x = float(sum) * __ldg(a_scale + t) * __ldg(w_scale + (e - t * f));
  put(out + e, lost ? __uint_as_float(0x7fffffffu) : x);
}

int64_t tiles_of(int64_t n, int64_t of) { return (n + of - 1) / of; }

// How a product is cut: tokens of a tile (0: the few rows' kernel), and parts of its contraction.
struct Cut {
  int tokens, splits;
};
constexpr int kPairs = 74;
Cut cut_of(int64_t m, int64_t k, int64_t f) {
  // Up to four rows of short contractions (three rows of 1,024 x 4,096 3.9 us, by tiles 5.4, eight 7.1 and 5.7; two of 8,192 x
  // 8,192 26 and 17).
  if (m == 1 || (m <= 4 && k <= 2048 && m * k * f <= 1 << 24)) return {0, 1};
  // Else the form that an estimate finds shortest, in cycles: a pair's rounds of tiles, each its steps and 1,200 for its begin and
  // end, a step 520 for 256 tokens, whose products it waits for, and 400 for fewer, whose operands it waits for; joined parts
  // cost a launch, some 5 us, and their writing and reading. Over 22 shapes it takes the quickest of 28 forms or one within 10%
  // (300 x 1,000 x 2,720: 64 tokens 7.5 us, 128 8.6, 256 9.3; 1,024 x 1,024 x 4,096: 256 tokens 9.0, 128 10.5, 64 12.8; 100 x
  // 8,192 x 300: 64 tokens in 8 parts 8.7 us, whole 17; 64 x 8,192 x 8,192: whole 17.9, in two parts 19.9).
  const int64_t steps = tiles_of(k, kStepBytes);
  Cut best{};
  double least = 0;
  for (int tokens = 32; tokens <= 256; tokens *= 2) {
    const int64_t tiles = tiles_of(m, tokens) * tiles_of(f, 2 * kChannelsEach);
    for (int most = 1; most <= 16 && most <= steps; most *= 2) {
      const int64_t split_steps = tiles_of(steps, most);
      const int splits = int(tiles_of(steps, split_steps));  // each with a step at least
      const int64_t rounds = tiles_of(tiles * splits, kPairs);
      const double step = tokens == 256 ? 520 : 400;
      double cycles = double(rounds) * (double(split_steps) * step + 1200);
      if (splits > 1) cycles += 10000 + double(m) * f * splits * 8 / 2500;
      if (best.tokens == 0 || cycles < least) best = {tokens, splits}, least = cycles;
    }
  }
  return best;
}

template <typename T, int kTokens, bool kWide = false>
int tiles(const Int8Product& q, int splits, void* scratch, cudaStream_t s) {
  using C = Int8Tile<kTokens, kWide>;
  Int8Tiles p{};
  p.m = q.m, p.f = q.f, p.a_scale = q.a_scale, p.w_scale = q.w_scale, p.out = q.out;
  p.splits = splits, p.parts = splits > 1 ? static_cast<int*>(scratch) : nullptr;
  const int64_t items = tiles_of(q.m, kTokens) * tiles_of(q.f, 2 * kChannelsEach) * splits;
  if (items > 0x7fff0000) return RLENV_EINVAL;
  p.token_tiles = int(tiles_of(q.m, kTokens)), p.channel_tiles = int(tiles_of(q.f, 2 * kChannelsEach));
  p.steps = int(tiles_of(q.k, kStepBytes)), p.split_steps = int(tiles_of(p.steps, splits));
  if (const int rc = bw::tile_map(&p.a, q.a, q.k, q.m, 1, q.a_pitch, C::kHalf, true)) return rc;
  if (const int rc = bw::tile_map(&p.w, q.w, q.k, q.f, 1, q.w_pitch, kChannelsEach, true)) return rc;
  if constexpr (kWide)
    if (const int rc = bw::result_map(&p.result, q.out, q.f, q.m, sizeof(T) == 4)) return rc;
  int dev = 0, sms = 0;
  if (cudaError_t e = cudaGetDevice(&dev)) return int(e);
  if (cudaError_t e = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev)) return int(e);
  if (cudaError_t e = cudaFuncSetAttribute(tile_kernel<T, kTokens, kWide>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmem))
    return int(e);
  const int grid = 2 * int(items < sms / 2 ? items : sms / 2);
  tile_kernel<T, kTokens, kWide><<<grid, C::kThreads, C::kSmem, s>>>(p, int(items));
  if (const int rc = launch_status(); rc || splits == 1) return rc;
  add_parts_kernel<T><<<grid_for(q.m * q.f, 256), 256, 0, s>>>(p.parts, splits, q.m, q.f, q.a_scale, q.w_scale,
                                                               static_cast<T*>(q.out));
  return launch_status();
}

template <typename T, int kRows, int kChannels, int kAhead>
int few_rows(const Int8Product& p, cudaStream_t s) {
  few_rows_kernel<T, kRows, kChannels, kAhead><<<unsigned((p.f + 4 * kChannels - 1) / (4 * kChannels)), 128, 0, s>>>(p);
  return launch_status();
}

template <typename T>
int product(const Int8Product& p, void* scratch, cudaStream_t s) {
  const Cut cut = cut_of(p.m, p.k, p.f);
  const bool on_lines = p.f * sizeof(T) % 16 == 0 && reinterpret_cast<uintptr_t>(p.out) % 16 == 0;
  if (cut.tokens == 256 && cut.splits == 1 && on_lines) return tiles<T, 256, true>(p, 1, scratch, s);
  if (cut.tokens == 256) return tiles<T, 256>(p, cut.splits, scratch, s);
  if (cut.tokens == 128) return tiles<T, 128>(p, cut.splits, scratch, s);
  if (cut.tokens == 64) return tiles<T, 64>(p, cut.splits, scratch, s);
  if (cut.tokens == 32) return tiles<T, 32>(p, cut.splits, scratch, s);
  if (p.m == 1) return few_rows<T, 1, 2, 2>(p, s);
  if (p.m == 2) return few_rows<T, 2, 4, 2>(p, s);
  return few_rows<T, 4, 4, 2>(p, s);
}

// The tiles' indices are 32-bit ones, a tensor copy's strides below 2^40 bytes.
bool int8_sizes(int64_t m, int64_t k, int64_t f) {
  return m >= 0 && f >= 0 && k >= 1 && k <= 131071 && m < (int64_t(1) << 31) - 256 && f < (int64_t(1) << 31) - 256;
}
bool on_boundary(const void* p, int size) { return p && reinterpret_cast<uintptr_t>(p) % size == 0; }

}  // namespace
}  // namespace rlenv

extern "C" {

int64_t rlenv_int8_linear_scratch_bytes(int64_t m, int64_t k, int64_t f) {
  using namespace rlenv;
  if (!int8_sizes(m, k, f)) return RLENV_EINVAL;
  if (m == 0 || f == 0) return 0;
  const Cut cut = cut_of(m, k, f);
  return cut.splits > 1 ? m * f * cut.splits * 4 : 0;
}

int rlenv_int8_linear_forward(int dtype, int64_t m, int64_t k, int64_t f, const int8_t* a, int64_t a_pitch,
                              const float* a_scale, const int8_t* w, int64_t w_pitch, const float* w_scale, void* out,
                              void* scratch, int64_t scratch_bytes, void* stream) {
  using namespace rlenv;
  if ((dtype != RLENV_F32 && dtype != RLENV_BF16) || !int8_sizes(m, k, f) || a_pitch < k || w_pitch < k || a_pitch % 16 ||
      w_pitch % 16 || a_pitch >= (int64_t(1) << 40) || w_pitch >= (int64_t(1) << 40))
    return RLENV_EINVAL;
  if (m == 0 || f == 0) return RLENV_OK;
  if (!on_boundary(a, 16) || !on_boundary(w, 16) || !on_boundary(a_scale, 4) || !on_boundary(w_scale, 4) ||
      !on_boundary(out, dtype == RLENV_F32 ? 4 : 2) ||
      !scratch_holds(scratch, scratch_bytes, rlenv_int8_linear_scratch_bytes(m, k, f)))
    return RLENV_EINVAL;
  const Int8Product p{m, k, f, a, w, a_pitch, w_pitch, a_scale, w_scale, out};
  return dtype == RLENV_F32 ? product<float>(p, scratch, as_stream(stream)) : product<__nv_bfloat16>(p, scratch, as_stream(stream));
}

int rlenv_int8_linear_status(unsigned int* gave_up, int clear) {
  using namespace rlenv;
  if (!gave_up) return RLENV_EINVAL;
  *gave_up = 0;
  return bw::read_given_up(gave_up, clear != 0);
}

}  // extern "C"
