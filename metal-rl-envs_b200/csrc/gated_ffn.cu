// Gated feed-forward block: h = act(x Wg) * (x Wu) for x (M, K) and weights (K, F), and its
// gradient. With g = x Wg, u = x Wu and the gradient dh of h,
//     dg = dh u act'(g),   du = dh act(g),
//     dx = dg Wg' + du Wu',   dWg = x' dg,   dWu = x' du.
// The backward pass forms g and u again from x instead of keeping them: 2 M F values less to
// store and read, and no rounding of g and u to the inputs' type.
//
// The products run on one kernel, product_kernel, on pairs of SMs: tiles of 2 x 128 rows on the tensor
// cores (tcgen05, cta_group::2), operands brought by tensor copies (TMA) into rings of shared memory
// buffers, two accumulators in tensor memory so that a tile's epilogue runs under the next one's products.
// A pair reads a 256 x 256 tile's operands once between its two SMs, 64 bytes a clock for each; with
// 128 x 256 tiles on single SMs it was 96, more than L2 gives, and the tensor cores ran at 56%.
// float32 operands are sums of three bfloat16 planes (8 + 8 + 8 bits of mantissa), laid out by
// pack_kernel; a product of two is six products of planes, the three below 2^-24 left out.
#include <cuda_bf16.h>

#include "blackwell.cuh"

namespace rlenv {
namespace {

enum Activation { kSilu = 0, kGelu = 1 };

// act(g) and act'(g): silu g / (1 + e^-g), or gelu g Phi(g) with the exact normal distribution. For
// bfloat16 results the fast exponential and division, good to 2^-20, are enough.
template <bool kFast>
RLENV_D void activate(int act, float g, float* y, float* slope) {
  if (act == kSilu) {
    const float s = kFast ? __fdividef(1.0f, 1.0f + __expf(-g)) : 1.0f / (1.0f + expf(-g));
    *y = g * s;
    *slope = s * (1.0f + g * (1.0f - s));
  } else {
    const float cdf = 0.5f * erfcf(-0.70710678f * g);
    *y = g * cdf;
    *slope = cdf + g * (0.39894228f * (kFast ? __expf(-0.5f * g * g) : expf(-0.5f * g * g)));
  }
}

// ---- operands ------------------------------------------------------------------------------------

// Planes of a (rows, cols) array as bfloat16 (planes, rows, pitch), pitch a multiple of 8: for float32
// the three whose sum it is, for bfloat16 a copy (rows that are not on 16-byte boundaries).
template <typename T, int kPlanes>
__global__ void __launch_bounds__(256)
pack_kernel(const T* __restrict__ from, int64_t rows, int64_t cols, int64_t pitch, __nv_bfloat16* __restrict__ to) {
  const int64_t pairs = pitch / 2, e = int64_t(blockIdx.x) * 256 + threadIdx.x;
  if (e >= rows * pairs) return;
  const int64_t r = e / pairs, c = e % pairs * 2;
  float lo = c < cols ? float(from[r * cols + c]) : 0.0f, hi = c + 1 < cols ? float(from[r * cols + c + 1]) : 0.0f;
#pragma unroll
  for (int q = 0; q < kPlanes; ++q) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
    *reinterpret_cast<__nv_bfloat162*>(to + (q * rows + r) * pitch + c) = v;
    lo -= __low2float(v), hi -= __high2float(v);
  }
}

// ---- the product kernel ---------------------------------------------------------------------------

enum Op { kForward, kGates, kGradients };  // h; dg and du; dx, dWg and dWu

constexpr int kRows = 128;       // of a tile, in each block of a pair
constexpr int kStep = 64;        // of the contraction, a ring buffer's
constexpr int kProductThreads = 384;  // copies, products, two idle warps, eight warps of epilogue
constexpr int kEpilogueWarps = 8;
constexpr int kTmemColumns = 512;
constexpr int kStagePitch = 33;  // floats: a 32 x 32 tile is written by rows and read by columns, or the other
                                 // way round, without bank conflicts

template <typename T>
struct Tile {
  static constexpr bool kFloat = sizeof(T) == 4;
  static constexpr int kPlanes = kFloat ? 3 : 1;
  static constexpr int kPairs = kFloat ? 6 : 1;  // products of planes
  static constexpr int kCols = kFloat ? 128 : 256;
  static constexpr int kHalf = kCols / 2;        // columns of B in each block
  static constexpr int kABytes = kRows * kStep * 2;
  static constexpr int kRingBytes = kABytes + kHalf * kStep * 2;
  static constexpr int kStages = kFloat ? 7 : 5;
  static constexpr int kStageAt = kStages * kRingBytes;  // the epilogue's 32 x 32 tiles, one a warp
  // the ring starts on a 1,024-byte boundary
  static constexpr int kSmem = kStageAt + kEpilogueWarps * 32 * kStagePitch * 4 + 1024;
  // Steps of the contraction summed in tensor memory before the epilogue takes them out into registers
  // (float32 only). The tensor core truncates as it accumulates; rounded additions of short sums keep
  // float32 results at float32's error. Of the products of planes only the leading one, the last to be
  // formed, is large enough to need the short sums.
  static constexpr int kRun = 4, kSmallRun = 32;
};

struct Operands {
  CUtensorMap a, b0, b1;
};
struct alignas(64) Product {
  Operands in[2];         // kGradients: of dx, then of the weights' gradients; else the first
  int64_t m, k, f;
  int act;
  // Tiles: of h or the gates; of dx and of both weights.
  int row_tiles, col_tiles, weight_rows, weight_cols;
  int splits, split_blocks;  // of the contraction over tokens in the weights' gradients
  const void* dh;            // kGates
  void *out, *dwg, *dwu;     // h or dx; the weights' gradients
  float* parts;              // (splits, 2, K, F) where splits > 1
  __nv_bfloat16* gates;      // (plane, dg or du, M, pitch)
  int64_t pitch;
};

// Tiles are taken in bands of kBand rows of tiles, column by column, so that those in flight share
// operands that lie in L2.
constexpr int kBand = 8;

// A tile of work: columns from c0, rows from row tile `row`, a contraction over `blocks` steps of each of
// `segs` segments from block k0.
struct Work {
  bool weights;
  int weight, split, row, c0, k0, blocks, segs;
};
template <typename T, int kOp>
RLENV_D Work work_of(const Product& p, int item) {
  Work w{};
  int rows = p.row_tiles, cols = p.col_tiles;
  w.segs = 1;
  if constexpr (kOp == kGradients) {
    // the weights' longer contractions first
    const int per = p.weight_rows * p.weight_cols;
    w.weights = item < per * p.splits;
    if (w.weights) {
      w.split = item / per, item %= per;
      rows = p.weight_rows, cols = p.weight_cols;
      w.k0 = w.split * p.split_blocks;
      w.blocks = min(p.split_blocks, int((p.m + kStep - 1) / kStep) - w.k0);
    } else {
      item -= per * p.splits;
      w.segs = 2, w.blocks = int((p.f + kStep - 1) / kStep);
    }
  } else {
    w.blocks = int((p.k + kStep - 1) / kStep);
  }
  const int per = kBand * cols, band = item / per, in = item % per;
  const int high = min(kBand, rows - band * kBand);
  w.row = band * kBand + in % high;
  int col = in / high;
  if (w.weights && col >= cols / 2) w.weight = 1, col -= cols / 2;
  w.c0 = col * (kOp == kGradients ? Tile<T>::kCols : Tile<T>::kHalf);
  return w;
}

// What a step multiplies: planes a and b, the small products first; segment; block of the contraction.
struct Step {
  int a, b, seg, k;
};
template <typename T>
RLENV_D Step step_of(const Work& w, int it) {
  const int per = w.segs * w.blocks, pair = it / per, in = it % per;
  Step s{0, 0, in / w.blocks, w.k0 + in % w.blocks};
  if (Tile<T>::kFloat) {
    switch (pair) {
      case 0: s.a = 0, s.b = 2; break;
      case 1: s.a = 2, s.b = 0; break;
      case 2: s.a = 1, s.b = 1; break;
      case 3: s.a = 0, s.b = 1; break;
      case 4: s.a = 1, s.b = 0; break;
      default: break;
    }
  }
  return s;
}
// Whether the accumulator is handed over after step `it` of `steps`.
template <typename T>
RLENV_D bool run_ends(int it, int steps) {
  if (it + 1 == steps) return true;
  if (!Tile<T>::kFloat) return false;
  const int small = steps / Tile<T>::kPairs * (Tile<T>::kPairs - 1);
  if (it + 1 <= small) return it + 1 == small || (it + 1) % Tile<T>::kSmallRun == 0;
  return (it + 1 - small) % Tile<T>::kRun == 0;
}

// A warp's 32 x 32 tile between registers (a row a lane) and an array (row pitch `pitch`), rows and
// columns past the ends left out, through shared memory so that global accesses run along rows.
template <typename T>
RLENV_D void store_tile(T* to, int64_t pitch, int rows, int cols, const float (&v)[32], float* stage) {
  const int lane = threadIdx.x & 31;
  __syncwarp();
#pragma unroll
  for (int i = 0; i < 32; ++i) stage[lane * kStagePitch + i] = v[i];
  __syncwarp();
  if (cols >= 32 && (reinterpret_cast<uintptr_t>(to) | uintptr_t(pitch * sizeof(T))) % (4 * sizeof(T)) == 0) {
    const int c = lane % 8 * 4;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int r = 4 * i + lane / 8;
      const float* s = stage + r * kStagePitch + c;
      if (r < rows) {
        if constexpr (sizeof(T) == 2) {
          const __nv_bfloat162 lo = __floats2bfloat162_rn(s[0], s[1]), hi = __floats2bfloat162_rn(s[2], s[3]);
          *reinterpret_cast<uint2*>(to + r * pitch + c) =
              make_uint2(*reinterpret_cast<const uint32_t*>(&lo), *reinterpret_cast<const uint32_t*>(&hi));
        } else {
          *reinterpret_cast<float4*>(to + r * pitch + c) = make_float4(s[0], s[1], s[2], s[3]);
        }
      }
    }
  } else {
#pragma unroll 8
    for (int r = 0; r < 32; ++r)
      if (r < rows && lane < cols) to[r * pitch + lane] = T(stage[r * kStagePitch + lane]);
  }
}
template <typename T>
RLENV_D void load_tile(const T* from, int64_t pitch, int rows, int cols, float (&v)[32], float* stage) {
  const int lane = threadIdx.x & 31;
  __syncwarp();
  if (cols >= 32 && (reinterpret_cast<uintptr_t>(from) | uintptr_t(pitch * sizeof(T))) % (4 * sizeof(T)) == 0) {
    const int c = lane % 8 * 4;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int r = 4 * i + lane / 8;
      float4 x = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      if (r < rows) {
        if constexpr (sizeof(T) == 2) {
          const uint2 w = __ldg(reinterpret_cast<const uint2*>(from + r * pitch + c));
          x = make_float4(__uint_as_float(w.x << 16), __uint_as_float(w.x & 0xffff0000u), __uint_as_float(w.y << 16),
                          __uint_as_float(w.y & 0xffff0000u));
        } else {
          x = __ldg(reinterpret_cast<const float4*>(from + r * pitch + c));
        }
      }
      float* s = stage + r * kStagePitch + c;
      s[0] = x.x, s[1] = x.y, s[2] = x.z, s[3] = x.w;
    }
  } else {
#pragma unroll 8
    for (int r = 0; r < 32; ++r)
      stage[r * kStagePitch + lane] = r < rows && lane < cols ? float(from[r * pitch + lane]) : 0.0f;
  }
  __syncwarp();
#pragma unroll
  for (int i = 0; i < 32; ++i) v[i] = stage[lane * kStagePitch + i];
}

// A 32 x 32 piece of a tile's results: rows from r0, columns from c (of h, a weight or dx). v holds its
// values or gates, u its ups.
template <typename T, int kOp>
RLENV_D void finish(const Product& p, const Work& w, int64_t r0, int64_t c, float (&v)[32], float (&u)[32],
                    float* stage) {
  constexpr bool kFast = !Tile<T>::kFloat;
  if constexpr (kOp == kGradients) {
    const int64_t all_rows = w.weights ? p.k : p.m, all_cols = w.weights ? p.f : p.k;
    if (r0 >= all_rows || c >= all_cols) return;
    const int rows = int(min(int64_t(32), all_rows - r0)), cols = int(min(int64_t(32), all_cols - c));
    if (w.weights && p.splits > 1) {
      store_tile(p.parts + ((int64_t(w.split) * 2 + w.weight) * p.k + r0) * p.f + c, p.f, rows, cols, v, stage);
    } else {
      T* to = static_cast<T*>(w.weights ? (w.weight ? p.dwu : p.dwg) : p.out);
      store_tile(to + r0 * all_cols + c, all_cols, rows, cols, v, stage);
    }
  } else {
    if (r0 >= p.m || c >= p.f) return;
    const int rows = int(min(int64_t(32), p.m - r0)), cols = int(min(int64_t(32), p.f - c));
    if constexpr (kOp == kForward) {
#pragma unroll
      for (int i = 0; i < 32; ++i) {
        float y, slope;
        activate<kFast>(p.act, v[i], &y, &slope);
        v[i] = y * u[i];
      }
      store_tile(static_cast<T*>(p.out) + r0 * p.f + c, p.f, rows, cols, v, stage);
    } else {
      float d[32];
      load_tile(static_cast<const T*>(p.dh) + r0 * p.f + c, p.f, rows, cols, d, stage);
#pragma unroll
      for (int i = 0; i < 32; ++i) {
        float y, slope;
        activate<kFast>(p.act, v[i], &y, &slope);
        v[i] = d[i] * u[i] * slope;
        u[i] = d[i] * y;
      }
#pragma unroll 1
      for (int q = 0; q < Tile<T>::kPlanes; ++q) {
        __nv_bfloat16* to = p.gates + (2 * q * p.m + r0) * p.pitch + c;
        store_tile(to, p.pitch, rows, cols, v, stage);
        store_tile(to + p.m * p.pitch, p.pitch, rows, cols, u, stage);
        if (Tile<T>::kPlanes > 1) {
#pragma unroll
          for (int i = 0; i < 32; ++i) {
            v[i] -= __bfloat162float(__float2bfloat16_rn(v[i]));
            u[i] -= __bfloat162float(__float2bfloat16_rn(u[i]));
          }
        }
      }
    }
  }
}

template <typename T, int kOp>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kProductThreads, 1)
product_kernel(const __grid_constant__ Product p, int items) {
  using C = Tile<T>;
  constexpr bool kPaired = kOp != kGradients;  // half of a tile's columns are gates, half ups
  constexpr uint32_t kBox = 64 * kStep * 2;
  extern __shared__ unsigned char raw[];
  __shared__ __align__(8) uint64_t bars[2 * C::kStages + 4];
  __shared__ uint32_t tmem_slot;
  __shared__ int dead_flag;
  volatile int* const dead = &dead_flag;
  const uint32_t ring = (bw::shared_at(raw) + 1023) & ~1023u;
  const uint32_t full = bw::shared_at(bars), empty = full + 8 * C::kStages;
  const uint32_t summed = empty + 8 * C::kStages, taken = summed + 16;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = int(bw::cluster_rank());
  if (threadIdx.x == 0) {
    for (int i = 0; i < C::kStages; ++i) bw::barrier_init(full + 8 * i, 1), bw::barrier_init(empty + 8 * i, 1);
    for (int i = 0; i < 2; ++i) bw::barrier_init(summed + 8 * i, 1), bw::barrier_init(taken + 8 * i, 2 * kEpilogueWarps);
    dead_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 2) bw::tmem_alloc<kTmemColumns>(bw::shared_at(&tmem_slot));
  bw::fence_before();
  __syncthreads();
  bw::cluster_sync();
  bw::fence_after();
  const uint32_t tmem = tmem_slot;
  const int first = blockIdx.x / 2, stride = gridDim.x / 2;

  if (warp == 0) {
    if (lane == 0) {
      // Both blocks copy their rows of A and their columns of B; all bytes count at the first block's barrier.
      int stage = 0;
      uint32_t phase = 0, used = 0;  // used: stages that have been filled at least once
      bool ok = true;
      const uint32_t full_at = bw::in_block(full, 0);
      for (int item = first; item < items && ok; item += stride) {
        const Work w = work_of<T, kOp>(p, item);
        const Operands& in = p.in[kOp == kGradients && w.weights];
        const int r0 = (2 * w.row + rank) * kRows, steps = C::kPairs * w.segs * w.blocks;
        for (int it = 0; it < steps; ++it) {
          const Step s = step_of<T>(w, it);
          const int k0 = s.k * kStep;
          if (!(ok = bw::barrier_wait(empty + 8 * stage, phase ^ 1, dead))) break;
          if (rank == 0) bw::barrier_expect(full + 8 * stage, 2 * C::kRingBytes);
          const uint32_t bar = full_at + 8 * stage, a = ring + stage * C::kRingBytes, b = a + C::kABytes;
          if (kPaired) {  // A by rows of the contraction's axis; gates in the first block, ups in the second
            bw::copy_tile(a, &in.a, bar, k0, r0, s.a);
            for (int i = 0; i < C::kHalf / 64; ++i)
              bw::copy_tile(b + i * kBox, rank ? &in.b1 : &in.b0, bar, w.c0 + 64 * i, k0, s.b);
          } else if (w.weights) {
            for (int i = 0; i < kRows / 64; ++i) bw::copy_tile(a + i * kBox, &in.a, bar, r0 + 64 * i, k0, s.a);
            for (int i = 0; i < C::kHalf / 64; ++i)
              bw::copy_tile(b + i * kBox, &in.b0, bar, w.c0 + rank * C::kHalf + 64 * i, k0, 2 * s.b + w.weight);
          } else {
            bw::copy_tile(a, &in.a, bar, k0, r0, 2 * s.a + s.seg);
            bw::copy_tile(b, s.seg ? &in.b1 : &in.b0, bar, k0, w.c0 + rank * C::kHalf, s.b);
          }
          used |= 1u << stage;
          if (++stage == C::kStages) stage = 0, phase ^= 1;
        }
      }
      if (!ok && rank == 0) {  // the copies in flight land before the blocks may end
        int unused = 0;
        for (int i = 0; i < C::kStages; ++i)
          if (used >> i & 1) bw::barrier_wait(full + 8 * i, i < stage ? phase : phase ^ 1, &unused), unused = 0;
      }
    }
  } else if (warp == 1) {
    if (lane == 0 && rank == 0) {
      int stage = 0, buffer = 0;
      uint32_t phase = 0, buffer_phase = 0;
      bool ok = true;
      for (int item = first; item < items && ok; item += stride) {
        const Work w = work_of<T, kOp>(p, item);
        const int steps = C::kPairs * w.segs * w.blocks;
        const bool mn_a = w.weights, mn_b = kPaired || w.weights;
        const uint32_t kind = bw::product_kind(2 * kRows, C::kCols, mn_a, mn_b);
        bool fresh = true;
        for (int it = 0; it < steps; ++it) {
          if (fresh && !(ok = bw::barrier_wait(taken + 8 * buffer, buffer_phase ^ 1, dead))) break;
          if (!(ok = bw::barrier_wait(full + 8 * stage, phase, dead))) break;
          bw::fence_after();
          const uint32_t a = ring + stage * C::kRingBytes, b = a + C::kABytes;
#pragma unroll
          for (int k = 0; k < kStep / 16; ++k)
            bw::multiply(tmem + buffer * C::kCols, bw::operand(a + k * (mn_a ? 2048 : 32), mn_a, kBox),
                         bw::operand(b + k * (mn_b ? 2048 : 32), mn_b, kBox), kind, !(fresh && k == 0));
          bw::commit(empty + 8 * stage);
          fresh = run_ends<T>(it, steps);
          if (fresh) {
            bw::commit(summed + 8 * buffer);
            if (++buffer == 2) buffer = 0, buffer_phase ^= 1;
          }
          if (++stage == C::kStages) stage = 0, phase ^= 1;
        }
      }
    }
  } else if (warp >= 4) {
    const int quarter = warp & 3, half = (warp - 4) >> 2;
    float* const own_stage = reinterpret_cast<float*>(raw + (ring - bw::shared_at(raw)) + C::kStageAt) +
                             (warp - 4) * 32 * kStagePitch;
    constexpr int kMine = C::kCols / 2;  // columns of the accumulator that a thread reads
    int buffer = 0;
    uint32_t buffer_phase = 0;
    bool ok = true;
    const uint32_t taken_at = bw::in_block(taken, 0), lanes = uint32_t(32 * quarter) << 16;
    const auto take_next = [&] {
      bw::fence_before();
      __syncwarp();
      if (lane == 0) bw::barrier_arrive(taken_at + 8 * buffer);
      if (++buffer == 2) buffer = 0, buffer_phase ^= 1;
    };
    // Run j of 32 columns of this thread's; a paired tile's second half of runs are ups.
    const auto column = [&](int j) {
      return kPaired ? (j < kMine / 64 ? 0 : C::kHalf - kMine / 2) + half * (kMine / 2) + 32 * j : half * kMine + 32 * j;
    };
    for (int item = first; item < items; item += stride) {
      const Work w = work_of<T, kOp>(p, item);
      const int64_t r0 = int64_t(2 * w.row + rank) * kRows + 32 * quarter;
      if constexpr (C::kFloat) {
        const int steps = C::kPairs * w.segs * w.blocks;
        float sum[kMine / 32][32];
#pragma unroll
        for (int j = 0; j < kMine / 32; ++j)
#pragma unroll
          for (int i = 0; i < 32; ++i) sum[j][i] = 0.0f;
        for (int it = 0; it < steps; ++it) {
          if (!run_ends<T>(it, steps)) continue;
          ok = ok && bw::barrier_wait(summed + 8 * buffer, buffer_phase, dead);
          ok = __all_sync(0xffffffffu, ok);
          if (!ok) break;
          bw::fence_after();
#pragma unroll
          for (int j = 0; j < kMine / 32; ++j) {
            float v[32];
            bw::tmem_load32(v, tmem + lanes + buffer * C::kCols + column(j));
#pragma unroll
            for (int i = 0; i < 32; ++i) sum[j][i] += v[i];
          }
          take_next();
        }
        if (!ok) {  // a wait ran out: the results say so
#pragma unroll
          for (int j = 0; j < kMine / 32; ++j)
#pragma unroll
            for (int i = 0; i < 32; ++i) sum[j][i] = __uint_as_float(0x7fffffffu);
        }
        if constexpr (kPaired) {
          finish<T, kOp>(p, w, r0, w.c0 + column(0), sum[0], sum[1], own_stage);
        } else {
#pragma unroll
          for (int j = 0; j < kMine / 32; ++j)
            finish<T, kOp>(p, w, r0, w.c0 + column(j), sum[j], sum[j], own_stage);
        }
      } else {
        ok = ok && bw::barrier_wait(summed + 8 * buffer, buffer_phase, dead);
        ok = __all_sync(0xffffffffu, ok);
        bw::fence_after();
#pragma unroll 1
        for (int j = 0; j < (kPaired ? kMine / 64 : kMine / 32); ++j) {
          float v[32], u[32];
          if (ok) {
            bw::tmem_load32(v, tmem + lanes + buffer * C::kCols + column(j));
            if (kPaired) bw::tmem_load32(u, tmem + lanes + buffer * C::kCols + column(j + kMine / 64));
          } else {
#pragma unroll
            for (int i = 0; i < 32; ++i) v[i] = u[i] = __uint_as_float(0x7fffffffu);
          }
          finish<T, kOp>(p, w, r0, w.c0 + column(j), v, u, own_stage);
        }
        take_next();
      }
    }
  }
  __syncwarp();
  bw::fence_before();
  __syncthreads();
  bw::cluster_sync();
  bw::fence_after();
  if (warp == 2) bw::tmem_free<kTmemColumns>(tmem);
}

// The weights' gradients from the sums over runs of tokens.
template <typename T>
__global__ void __launch_bounds__(256)
add_parts_kernel(const float* __restrict__ parts, int splits, int64_t size, T* __restrict__ dwg, T* __restrict__ dwu) {
  const int64_t e = int64_t(blockIdx.x) * 256 + threadIdx.x;
  if (e >= 2 * size) return;
  float sum = 0.0f;
  for (int s = 0; s < splits; ++s) sum += __ldg(parts + s * 2 * size + e);
  (e < size ? dwg : dwu)[e < size ? e : e - size] = T(sum);
}

// ---- host ------------------------------------------------------------------------------------------

constexpr int64_t kMaxExtent = int64_t(1) << 31;

int check_ffn(int dtype, int act, int64_t m, int64_t k, int64_t f) {
  if (dtype != RLENV_F32 && dtype != RLENV_BF16) return RLENV_EINVAL;
  if (act != kSilu && act != kGelu) return RLENV_EINVAL;
  if (m < 0 || k < 0 || f < 0 || m >= kMaxExtent || k >= kMaxExtent || f >= kMaxExtent / 2) return RLENV_EINVAL;
  return RLENV_OK;
}

int64_t round_up(int64_t n, int64_t to) { return (n + to - 1) / to * to; }

// An operand (rows, cols): the caller's own array where tensor copies can read it, else its planes in scratch.
struct Operand {
  const __nv_bfloat16* base;
  int64_t rows, cols, pitch, slices;
  int map(CUtensorMap* to, int box_rows) const { return bw::tile_map(to, base, cols, rows, slices, pitch, box_rows); }
};

// Hands out scratch by 256 bytes; with base null it only counts.
struct Scratch {
  unsigned char* base;
  int64_t used;
  void* take(int64_t bytes) {
    void* p = base ? base + used : nullptr;
    used += round_up(bytes, 256);
    return p;
  }
};

// dtype's planes of (rows, cols) need packing: float32 always, bfloat16 where a row is no multiple of 16
// bytes. (A base off the 16-byte boundary is refused: the wrappers' tensors start on one.)
bool packs(int dtype, int64_t cols) { return dtype == RLENV_F32 || cols % 8 != 0; }
int64_t planes(int dtype) { return dtype == RLENV_F32 ? 3 : 1; }

struct Layout {  // scratch of a call
  void *x, *wg, *wu, *gates;
  float* parts;
  int splits, split_blocks;
  int64_t bytes;
};

constexpr int kPairsOfSms = 74;
constexpr int64_t kFewestBlocks = 8;

// The contraction over tokens of the weights' gradients is split where a tile of them would take longer
// than a pair of SMs' share of all the work: a small block's weights are a few tiles, each a sum over every
// token. The sums of each run of tokens are kept in float32 and added up in order.
void split_tokens(int dtype, int64_t m, int64_t k, int64_t f, Layout* l) {
  const int64_t wide = dtype == RLENV_F32 ? 128 : 256, high = 2 * kRows;
  const int64_t blocks = (m + kStep - 1) / kStep, tiles = (k + high - 1) / high * ((f + wide - 1) / wide) * 2;
  const int64_t dx = (m + high - 1) / high * ((k + wide - 1) / wide) * 2 * ((f + kStep - 1) / kStep);
  int64_t share = (tiles * blocks + dx) / kPairsOfSms;
  if (share < kFewestBlocks) share = kFewestBlocks;
  int64_t splits = (blocks + share - 1) / share;
  if (splits < 1) splits = 1;
  l->split_blocks = int((blocks + splits - 1) / splits);
  l->splits = int((blocks + l->split_blocks - 1) / l->split_blocks);
}
Layout lay_out(int dtype, int64_t m, int64_t k, int64_t f, bool backward, void* scratch) {
  Scratch s{static_cast<unsigned char*>(scratch), 0};
  Layout l{};
  const int64_t n = planes(dtype);
  if (packs(dtype, k)) l.x = s.take(n * m * round_up(k, 8) * 2);
  if (packs(dtype, f)) l.wg = s.take(n * k * round_up(f, 8) * 2), l.wu = s.take(n * k * round_up(f, 8) * 2);
  if (backward) {
    l.gates = s.take(2 * n * m * round_up(f, 8) * 2);
    if (m > 0 && k > 0 && f > 0) split_tokens(dtype, m, k, f, &l);
    if (l.splits > 1) l.parts = static_cast<float*>(s.take(int64_t(l.splits) * 2 * k * f * 4));
  }
  l.bytes = s.used;
  return l;
}

template <typename T>
int operand(const void* from, int64_t rows, int64_t cols, void* packed, cudaStream_t s, Operand* o) {
  constexpr int kPlanes = Tile<T>::kPlanes;
  if (!packed) {
    *o = {static_cast<const __nv_bfloat16*>(from), rows, cols, cols, 1};
    return RLENV_OK;
  }
  const int64_t pitch = round_up(cols, 8), pairs = rows * (pitch / 2);
  pack_kernel<T, kPlanes><<<unsigned((pairs + 255) / 256), 256, 0, s>>>(static_cast<const T*>(from), rows, cols, pitch,
                                                                       static_cast<__nv_bfloat16*>(packed));
  *o = {static_cast<const __nv_bfloat16*>(packed), rows, cols, pitch, kPlanes};
  return launch_status();
}

template <typename T, int kOp>
int run_product(const Product& p, cudaStream_t s) {
  using C = Tile<T>;
  const int64_t items = int64_t(p.row_tiles) * p.col_tiles + int64_t(p.weight_rows) * p.weight_cols * p.splits;
  if (items > 0x7fffffff) return RLENV_EINVAL;
  int dev = 0, sms = 0;
  if (cudaError_t e = cudaGetDevice(&dev)) return int(e);
  if (cudaError_t e = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev)) return int(e);
  if (cudaError_t e = cudaFuncSetAttribute(product_kernel<T, kOp>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmem))
    return int(e);
  const int grid = 2 * int(items < sms / 2 ? items : sms / 2);
  product_kernel<T, kOp><<<grid, kProductThreads, C::kSmem, s>>>(p, int(items));
  return launch_status();
}

int tile_count(int64_t n, int64_t of) { return int((n + of - 1) / of); }

template <typename T>
int ffn(const void* dh, const void* x, const void* wg, const void* wu, int64_t m, int64_t k, int64_t f, int act,
        void* out, void* dx, void* dwg, void* dwu, const Layout& l, cudaStream_t s) {
  using C = Tile<T>;
  Operand X, G, U;
  if (const int rc = operand<T>(x, m, k, l.x, s, &X)) return rc;
  if (const int rc = operand<T>(wg, k, f, l.wg, s, &G)) return rc;
  if (const int rc = operand<T>(wu, k, f, l.wu, s, &U)) return rc;
  Product p{};
  p.m = m, p.k = k, p.f = f, p.act = act, p.out = out, p.dh = dh;
  p.gates = static_cast<__nv_bfloat16*>(l.gates), p.pitch = round_up(f, 8);
  p.row_tiles = tile_count(m, 2 * kRows), p.col_tiles = tile_count(f, C::kHalf);
  if (const int rc = X.map(&p.in[0].a, kRows)) return rc;
  if (const int rc = G.map(&p.in[0].b0, 64)) return rc;
  if (const int rc = U.map(&p.in[0].b1, 64)) return rc;
  if (!dh) return run_product<T, kForward>(p, s);
  if (const int rc = run_product<T, kGates>(p, s)) return rc;
  const Operand D{p.gates, m, f, p.pitch, 2 * C::kPlanes};
  p.out = dx, p.dwg = dwg, p.dwu = dwu, p.parts = l.parts, p.splits = l.splits, p.split_blocks = l.split_blocks;
  p.col_tiles = tile_count(k, C::kCols);
  p.weight_rows = tile_count(k, 2 * kRows), p.weight_cols = 2 * tile_count(f, C::kCols);
  if (const int rc = D.map(&p.in[0].a, kRows)) return rc;
  if (const int rc = G.map(&p.in[0].b0, C::kHalf)) return rc;
  if (const int rc = U.map(&p.in[0].b1, C::kHalf)) return rc;
  if (const int rc = X.map(&p.in[1].a, 64)) return rc;
  if (const int rc = D.map(&p.in[1].b0, 64)) return rc;
  if (const int rc = run_product<T, kGradients>(p, s)) return rc;
  if (l.splits == 1) return RLENV_OK;
  add_parts_kernel<T><<<grid_for(2 * k * f, 256), 256, 0, s>>>(l.parts, l.splits, k * f, static_cast<T*>(dwg),
                                                               static_cast<T*>(dwu));
  return launch_status();
}

bool off_boundary(const void* a, const void* b, const void* c) {
  return (reinterpret_cast<uintptr_t>(a) | reinterpret_cast<uintptr_t>(b) | reinterpret_cast<uintptr_t>(c)) % 16 != 0;
}

}  // namespace
}  // namespace rlenv

extern "C" {

int64_t rlenv_gated_ffn_scratch_bytes(int dtype, int64_t m, int64_t k, int64_t f, int backward) {
  using namespace rlenv;
  if (check_ffn(dtype, 0, m, k, f) != RLENV_OK) return -1;
  return lay_out(dtype, m, k, f, backward != 0, nullptr).bytes;
}

int rlenv_gated_ffn_forward(int dtype, int activation, int64_t m, int64_t k, int64_t f, const void* x,
                            const void* w_gate, const void* w_up, void* out, void* scratch, int64_t scratch_bytes,
                            void* stream) {
  using namespace rlenv;
  if (const int rc = check_ffn(dtype, activation, m, k, f)) return rc;
  if (m == 0 || f == 0) return RLENV_OK;
  if (k == 0) return out ? int(cudaMemsetAsync(out, 0, size_t(m) * f * (dtype == RLENV_F32 ? 4 : 2), as_stream(stream)))
                         : RLENV_EINVAL;
  if (!out || !x || !w_gate || !w_up || off_boundary(x, w_gate, w_up)) return RLENV_EINVAL;
  const Layout l = lay_out(dtype, m, k, f, false, scratch);
  if (!scratch_holds(scratch, scratch_bytes, l.bytes)) return RLENV_EINVAL;
  const cudaStream_t s = as_stream(stream);
  return dtype == RLENV_F32
             ? ffn<float>(nullptr, x, w_gate, w_up, m, k, f, activation, out, nullptr, nullptr, nullptr, l, s)
             : ffn<__nv_bfloat16>(nullptr, x, w_gate, w_up, m, k, f, activation, out, nullptr, nullptr, nullptr, l, s);
}

int rlenv_gated_ffn_backward(int dtype, int activation, int64_t m, int64_t k, int64_t f, const void* grad_out,
                             const void* x, const void* w_gate, const void* w_up, void* grad_x, void* grad_w_gate,
                             void* grad_w_up, void* scratch, int64_t scratch_bytes, void* stream) {
  using namespace rlenv;
  if (const int rc = check_ffn(dtype, activation, m, k, f)) return rc;
  if (m == 0 || k == 0 || f == 0) return RLENV_EINVAL;
  if (!grad_out || !x || !w_gate || !w_up || !grad_x || !grad_w_gate || !grad_w_up || off_boundary(x, w_gate, w_up))
    return RLENV_EINVAL;
  const Layout l = lay_out(dtype, m, k, f, true, scratch);
  if (!scratch_holds(scratch, scratch_bytes, l.bytes)) return RLENV_EINVAL;
  const cudaStream_t s = as_stream(stream);
  return dtype == RLENV_F32 ? ffn<float>(grad_out, x, w_gate, w_up, m, k, f, activation, nullptr, grad_x, grad_w_gate,
                                         grad_w_up, l, s)
                            : ffn<__nv_bfloat16>(grad_out, x, w_gate, w_up, m, k, f, activation, nullptr, grad_x,
                                                 grad_w_gate, grad_w_up, l, s);
}

}  // extern "C"
