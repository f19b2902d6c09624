// Gated feed-forward block: h = act(x Wg) * (x Wu) for x (M, K) and weights (K, F), and its
// gradient. With g = x Wg, u = x Wu and the gradient dh of h,
//     dg = dh u act'(g),   du = dh act(g),
//     dx = dg Wg' + du Wu',   dWg = x' dg,   dWu = x' du.
// The backward pass forms g and u again from x instead of keeping them: 2 M F values less to
// store and read, and no rounding of g and u to the inputs' type.
//
// All four products run on one kernel, product_kernel: tiles of 128 rows on the tensor cores
// (tcgen05), operands brought by tensor copies (TMA) into a ring of shared memory buffers, two
// accumulators in tensor memory so that one tile's epilogue runs under the next one's products.
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

enum Op { kForward, kGates, kInput, kWeights };  // h; dg and du; dx; dWg and dWu

constexpr int kRows = 128;       // of a tile
constexpr int kStep = 64;        // of the contraction, a ring buffer's
constexpr int kProductThreads = 384;  // copies, products, two idle warps, eight warps of epilogue
constexpr int kEpilogueWarps = 8;
constexpr int kTmemColumns = 512;

template <typename T>
struct Tile {
  static constexpr bool kFloat = sizeof(T) == 4;
  static constexpr int kPlanes = kFloat ? 3 : 1;
  static constexpr int kPairs = kFloat ? 6 : 1;  // products of planes
  static constexpr int kCols = kFloat ? 128 : 256;
  static constexpr int kStageBytes = (kRows + kCols) * kStep * 2;
  static constexpr int kStages = 196608 / kStageBytes;
  static constexpr int kSmem = kStages * kStageBytes + 1024;  // the ring starts on a 1,024-byte boundary
  // Steps of the contraction summed in tensor memory before the epilogue takes them out into registers
  // (0: all). The tensor core truncates as it accumulates; rounded additions of short sums keep float32
  // results at float32's error. Only the leading planes' product, the last to be formed, is large
  // enough to matter.
  static constexpr int kRun = kFloat ? 4 : 0, kSmallRun = 32;
};

struct alignas(64) Product {
  CUtensorMap a, b0, b1;
  int64_t rows, cols;     // of the result (cols: F for kForward, kGates; of one weight for kWeights)
  int64_t depth;          // of one contraction (kInput has two, over dg Wg' and du Wu')
  int row_tiles, col_tiles;
  int act;
  const void* dh;         // kGates
  void *out0, *out1;      // h; dx; dWg and dWu
  __nv_bfloat16* gates;   // kGates: (plane, dg or du, rows, pitch)
  int64_t pitch;
};

// Tiles are taken in bands of kBand rows of tiles, column by column, so that those in flight share
// operands that lie in L2.
constexpr int kBand = 16;
struct Place {
  int row, col;
};
RLENV_D Place place(const Product& p, int tile) {
  const int per = kBand * p.col_tiles, band = tile / per, in = tile % per;
  const int high = min(kBand, p.row_tiles - band * kBand);
  return {band * kBand + in % high, in / high};
}

// What a step of a tile's contraction multiplies: planes a and b (small products first), segment seg
// (kInput), block k of the contraction.
struct Step {
  int a, b, seg, k;
};
template <typename T, int kOp>
RLENV_D Step step_of(int it, int blocks) {
  constexpr int kSegs = kOp == kInput ? 2 : 1;
  const int pair = it / (kSegs * blocks), in = it % (kSegs * blocks);
  Step s{0, 0, in / blocks, in % blocks};
  if (Tile<T>::kPairs > 1) {
    switch (pair) {
      case 0: s.a = 0, s.b = 2; break;
      case 1: s.a = 2, s.b = 0; break;
      case 2: s.a = 1, s.b = 1; break;
      case 3: s.a = 0, s.b = 1; break;
      case 4: s.a = 1, s.b = 0; break;
      default: s.a = 0, s.b = 0;
    }
  }
  return s;
}
// Whether the accumulator is handed over after step `it` of `steps`.
template <typename T>
RLENV_D bool run_ends(int it, int steps) {
  if (it + 1 == steps) return true;
  if constexpr (!Tile<T>::kFloat) return false;
  const int small = steps / Tile<T>::kPairs * (Tile<T>::kPairs - 1);
  if (it + 1 <= small) return it + 1 == small || (it + 1) % Tile<T>::kSmallRun == 0;
  return (it + 1 - small) % Tile<T>::kRun == 0;
}

template <typename T>
RLENV_D float load_one(const T* p, int64_t i) { return float(p[i]); }

// n <= 32 values to consecutive places, by 16 bytes where the whole run is there and on the boundary.
template <typename T>
RLENV_D void store_run(T* to, const float (&v)[32], int n) {
  if constexpr (sizeof(T) == 2) {
    if (n >= 32 && reinterpret_cast<uintptr_t>(to) % 16 == 0) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        uint32_t w[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const __nv_bfloat162 x = __floats2bfloat162_rn(v[8 * i + 2 * j], v[8 * i + 2 * j + 1]);
          w[j] = *reinterpret_cast<const uint32_t*>(&x);
        }
        reinterpret_cast<uint4*>(to)[i] = make_uint4(w[0], w[1], w[2], w[3]);
      }
      return;
    }
  } else {
    if (n >= 32 && reinterpret_cast<uintptr_t>(to) % 16 == 0) {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        reinterpret_cast<float4*>(to)[i] = make_float4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]);
      return;
    }
  }
#pragma unroll
  for (int i = 0; i < 32; ++i)
    if (i < n) to[i] = T(v[i]);
}

template <typename T, int kOp>
__global__ void __launch_bounds__(kProductThreads, 1) product_kernel(const __grid_constant__ Product p) {
  using C = Tile<T>;
  constexpr bool kPaired = kOp == kForward || kOp == kGates;  // half a tile's columns are gates, half ups
  constexpr bool kMnA = kOp == kWeights, kMnB = kOp != kInput;
  constexpr int kSegs = kOp == kInput ? 2 : 1;
  constexpr uint32_t kABytes = kRows * kStep * 2, kHalfB = C::kCols / 2 * kStep * 2, kBox = 64 * kStep * 2;
  extern __shared__ unsigned char raw[];
  __shared__ __align__(8) uint64_t bars[2 * C::kStages + 4];
  __shared__ uint32_t tmem_slot;
  __shared__ int dead_flag;
  volatile int* const dead = &dead_flag;
  const uint32_t ring = (bw::shared_at(raw) + 1023) & ~1023u;
  const uint32_t full = bw::shared_at(bars), empty = full + 8 * C::kStages;
  const uint32_t summed = empty + 8 * C::kStages, taken = summed + 16;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int i = 0; i < C::kStages; ++i) bw::barrier_init(full + 8 * i, 1), bw::barrier_init(empty + 8 * i, 1);
    for (int i = 0; i < 2; ++i) bw::barrier_init(summed + 8 * i, 1), bw::barrier_init(taken + 8 * i, kEpilogueWarps);
    dead_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 2) bw::tmem_alloc<kTmemColumns>(bw::shared_at(&tmem_slot));
  bw::fence_before();
  __syncthreads();
  bw::fence_after();
  const uint32_t tmem = tmem_slot;
  const int tiles = p.row_tiles * p.col_tiles;
  const int blocks = int((p.depth + kStep - 1) / kStep), steps = C::kPairs * kSegs * blocks;

  if (warp == 0) {
    if (lane == 0) {
      bw::prefetch_map(&p.a);
      bw::prefetch_map(&p.b0);
      if (kOp != kWeights) bw::prefetch_map(&p.b1);
      int stage = 0;
      uint32_t phase = 0, used = 0;  // used: stages that have been filled at least once
      bool ok = true;
      for (int tile = blockIdx.x; tile < tiles && ok; tile += gridDim.x) {
        const Place at = place(p, tile);
        const int half_cols = p.col_tiles / 2;
        const int weight = kOp == kWeights && at.col >= half_cols;
        const int r0 = at.row * kRows;
        const int c0 = (kOp == kWeights ? at.col - weight * half_cols : at.col) * (kPaired ? C::kCols / 2 : C::kCols);
        for (int it = 0; it < steps; ++it) {
          const Step s = step_of<T, kOp>(it, blocks);
          const int k0 = s.k * kStep;
          if (!(ok = bw::barrier_wait(empty + 8 * stage, phase ^ 1, dead))) break;
          const uint32_t bar = full + 8 * stage, a = ring + stage * C::kStageBytes, b = a + kABytes;
          bw::barrier_expect(bar, C::kStageBytes);
          if (kMnA) {
            for (int i = 0; i < kRows / 64; ++i) bw::copy_tile(a + i * kBox, &p.a, bar, r0 + 64 * i, k0, s.a);
          } else {
            bw::copy_tile(a, &p.a, bar, k0, r0, kOp == kInput ? 2 * s.a + s.seg : s.a);
          }
          if (kPaired) {
            for (int i = 0; i < C::kCols / 128; ++i) {
              bw::copy_tile(b + i * kBox, &p.b0, bar, c0 + 64 * i, k0, s.b);
              bw::copy_tile(b + kHalfB + i * kBox, &p.b1, bar, c0 + 64 * i, k0, s.b);
            }
          } else if (kOp == kInput) {
            for (int i = 0; i < C::kCols / 128; ++i)
              bw::copy_tile(b + i * 2 * kBox, s.seg ? &p.b1 : &p.b0, bar, k0, c0 + 128 * i, s.b);
          } else {
            for (int i = 0; i < C::kCols / 64; ++i)
              bw::copy_tile(b + i * kBox, &p.b0, bar, c0 + 64 * i, k0, 2 * s.b + weight);
          }
          used |= 1u << stage;
          if (++stage == C::kStages) stage = 0, phase ^= 1;
        }
      }
      if (!ok) {  // the copies in flight land before the block may end
        int unused = 0;
        for (int i = 0; i < C::kStages; ++i)
          if (used >> i & 1) {
            const uint32_t last = i < stage ? phase : phase ^ 1;
            bw::barrier_wait(full + 8 * i, last, &unused);
            unused = 0;
          }
      }
    }
  } else if (warp == 1) {
    if (lane == 0) {
      constexpr uint32_t kind = bw::product_kind(kRows, C::kCols, kMnA, kMnB);
      int stage = 0, buffer = 0;
      uint32_t phase = 0, buffer_phase = 0;
      bool ok = true;
      for (int tile = blockIdx.x; tile < tiles && ok; tile += gridDim.x) {
        bool fresh = true;
        for (int it = 0; it < steps; ++it) {
          if (fresh && !(ok = bw::barrier_wait(taken + 8 * buffer, buffer_phase ^ 1, dead))) break;
          if (!(ok = bw::barrier_wait(full + 8 * stage, phase, dead))) break;
          bw::fence_after();
          const uint32_t a = ring + stage * C::kStageBytes, b = a + kABytes;
#pragma unroll
          for (int k = 0; k < kStep / 16; ++k)
            bw::multiply(tmem + buffer * C::kCols, bw::operand(a + k * (kMnA ? 2048 : 32), kMnA, kBox),
                         bw::operand(b + k * (kMnB ? 2048 : 32), kMnB, kBox), kind, !(fresh && k == 0));
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
    constexpr int kMine = C::kCols / 2;  // columns of the accumulator that a thread reads
    int buffer = 0;
    uint32_t buffer_phase = 0;
    bool ok = true;
    for (int tile = blockIdx.x; tile < tiles; tile += gridDim.x) {
      const Place at = place(p, tile);
      const int half_cols = p.col_tiles / 2;
      const int weight = kOp == kWeights && at.col >= half_cols;
      const int64_t row = int64_t(at.row) * kRows + 32 * quarter + lane;
      const int64_t c0 = int64_t(kOp == kWeights ? at.col - weight * half_cols : at.col) *
                         (kPaired ? C::kCols / 2 : C::kCols);
      // Columns of the accumulator by 32: run j of this thread's. A paired tile's second half of runs are ups.
      const auto column = [&](int j) {
        return kPaired ? (j < kMine / 64 ? 0 : C::kCols / 2 - kMine / 2) + half * (kMine / 2) + 32 * j : half * kMine + 32 * j;
      };
      const auto finish = [&](float (&v)[32], float (&u)[32], int j) {
        const int64_t c = c0 + column(j);
        if (row >= p.rows || c >= p.cols) return;
        const int n = p.cols - c < 32 ? int(p.cols - c) : 32;
        if constexpr (kOp == kForward) {
#pragma unroll
          for (int i = 0; i < 32; ++i) {
            float y, slope;
            activate<!C::kFloat>(p.act, v[i], &y, &slope);
            v[i] = y * u[i];
          }
          store_run(static_cast<T*>(p.out0) + row * p.cols + c, v, n);
        } else if constexpr (kOp == kGates) {
          const T* dh = static_cast<const T*>(p.dh) + row * p.cols + c;
#pragma unroll
          for (int i = 0; i < 32; ++i) {
            float y, slope;
            activate<!C::kFloat>(p.act, v[i], &y, &slope);
            const float d = i < n ? load_one(dh, i) : 0.0f;
            v[i] = d * u[i] * slope;
            u[i] = d * y;
          }
          for (int q = 0; q < C::kPlanes; ++q) {
            __nv_bfloat16* to = p.gates + (2 * q * p.rows + row) * p.pitch + c;
            store_run(to, v, n);
            store_run(to + p.rows * p.pitch, u, n);
            if (C::kPlanes > 1) {
#pragma unroll
              for (int i = 0; i < 32; ++i) {
                v[i] -= __bfloat162float(__float2bfloat16_rn(v[i]));
                u[i] -= __bfloat162float(__float2bfloat16_rn(u[i]));
              }
            }
          }
        } else {
          T* out = static_cast<T*>(kOp == kWeights && weight ? p.out1 : p.out0);
          store_run(out + row * p.cols + c, v, n);
        }
      };
      const uint32_t lanes = uint32_t(32 * quarter) << 16;
      if constexpr (C::kFloat) {
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
          bw::fence_before();
          __syncwarp();
          if (lane == 0) bw::barrier_arrive(taken + 8 * buffer);
          if (++buffer == 2) buffer = 0, buffer_phase ^= 1;
        }
        if (!ok) {
#pragma unroll
          for (int j = 0; j < kMine / 32; ++j)
#pragma unroll
            for (int i = 0; i < 32; ++i) sum[j][i] = __uint_as_float(0x7fffffffu);
        }
        if constexpr (kPaired) {
          finish(sum[0], sum[1], 0);
        } else {
#pragma unroll
          for (int j = 0; j < kMine / 32; ++j) finish(sum[j], sum[j], j);
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
          finish(v, u, j);
        }
        bw::fence_before();
        __syncwarp();
        if (lane == 0) bw::barrier_arrive(taken + 8 * buffer);
        if (++buffer == 2) buffer = 0, buffer_phase ^= 1;
      }
    }
  }
  __syncwarp();
  bw::fence_before();
  __syncthreads();
  bw::fence_after();
  if (warp == 2) bw::tmem_free<kTmemColumns>(tmem);
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
  int64_t bytes;
};
Layout lay_out(int dtype, int64_t m, int64_t k, int64_t f, bool backward, void* scratch) {
  Scratch s{static_cast<unsigned char*>(scratch), 0};
  Layout l{};
  const int64_t n = planes(dtype);
  if (packs(dtype, k)) l.x = s.take(n * m * round_up(k, 8) * 2);
  if (packs(dtype, f)) l.wg = s.take(n * k * round_up(f, 8) * 2), l.wu = s.take(n * k * round_up(f, 8) * 2);
  if (backward) l.gates = s.take(2 * n * m * round_up(f, 8) * 2);
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
int run_product(Product& p, cudaStream_t s) {
  using C = Tile<T>;
  constexpr bool kPaired = kOp == kForward || kOp == kGates;
  const int64_t wide = kPaired ? C::kCols / 2 : C::kCols;
  const int64_t rt = (p.rows + kRows - 1) / kRows, ct = (p.cols + wide - 1) / wide * (kOp == kWeights ? 2 : 1);
  if (rt * ct > 0x7fffffff) return RLENV_EINVAL;
  p.row_tiles = int(rt), p.col_tiles = int(ct);
  int dev = 0, sms = 0;
  if (cudaError_t e = cudaGetDevice(&dev)) return int(e);
  if (cudaError_t e = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev)) return int(e);
  if (cudaError_t e = cudaFuncSetAttribute(product_kernel<T, kOp>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmem))
    return int(e);
  const int grid = int(rt * ct < sms ? rt * ct : sms);
  product_kernel<T, kOp><<<grid, kProductThreads, C::kSmem, s>>>(p);
  return launch_status();
}

template <typename T>
int ffn(const void* dh, const void* x, const void* wg, const void* wu, int64_t m, int64_t k, int64_t f, int act,
        void* out, void* dx, void* dwg, void* dwu, const Layout& l, cudaStream_t s) {
  Operand X, G, U;
  if (const int rc = operand<T>(x, m, k, l.x, s, &X)) return rc;
  if (const int rc = operand<T>(wg, k, f, l.wg, s, &G)) return rc;
  if (const int rc = operand<T>(wu, k, f, l.wu, s, &U)) return rc;
  Product p{};
  p.rows = m, p.cols = f, p.depth = k, p.act = act, p.out0 = out, p.dh = dh;
  p.gates = static_cast<__nv_bfloat16*>(l.gates), p.pitch = round_up(f, 8);
  if (const int rc = X.map(&p.a, kRows)) return rc;
  if (const int rc = G.map(&p.b0, 64)) return rc;
  if (const int rc = U.map(&p.b1, 64)) return rc;
  if (!dh) return run_product<T, kForward>(p, s);
  if (const int rc = run_product<T, kGates>(p, s)) return rc;
  const Operand D{p.gates, m, f, p.pitch, 2 * Tile<T>::kPlanes};
  Product q{};
  q.rows = m, q.cols = k, q.depth = f, q.out0 = dx;
  if (const int rc = D.map(&q.a, kRows)) return rc;
  if (const int rc = G.map(&q.b0, 128)) return rc;
  if (const int rc = U.map(&q.b1, 128)) return rc;
  if (const int rc = run_product<T, kInput>(q, s)) return rc;
  Product w{};
  w.rows = k, w.cols = f, w.depth = m, w.out0 = dwg, w.out1 = dwu;
  if (const int rc = X.map(&w.a, 64)) return rc;
  if (const int rc = D.map(&w.b0, 64)) return rc;
  return run_product<T, kWeights>(w, s);
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
