// Gated feed-forward block: h = act(x Wg) * (x Wu) for x (M, K) and weights (K, F), and its
// gradient. With g = x Wg, u = x Wu and the gradient dh of h,
//     dg = dh u act'(g),   du = dh act(g),
//     dx = dg Wg' + du Wu',   dWg = x' dg,   dWu = x' du.
// dg and du pass through the inputs' type on their way into the last three products, for bfloat16 through its 8
// bits, as in a program that keeps them as tensors: a second plane would double those products' time. Against 64
// bits the gradients of 8,192 x 1,024 x 2,720 are off by 0.0023, with 32-bit dg and du by 0.0017. (Few rows keep
// them in 32.)
// The backward pass forms g and u again from x instead of keeping them: 2 M F values less to
// store and read, and no rounding of g and u to the inputs' type.
//
// The products run on one kernel, product_kernel, on pairs of SMs: tiles of 2 x 128 rows on the tensor
// cores (tcgen05, cta_group::2), operands brought by tensor copies (TMA) into rings of shared memory
// buffers, two accumulators in tensor memory so that a tile's epilogue runs under the next one's products.
// A pair reads a 256 x 256 tile's operands once between its two SMs, 64 bytes a clock for each, where single
// SMs with tiles of 128 x 256 read 96.
//
// Measured: a step of 64 of the contraction takes a pair 515 cycles of at least 512 in bfloat16, and three such in
// float32 (six products of half as wide a tile), so that the clock under the power limit is what is left of
// long contractions: 16,384 x 1,024 x 4,096 forward 171 us in a short run (1.61 PFLOP/s), 211 us sustained;
// float32 4,330 x 881 x 1,780 forward 104 us. Where the contraction is short the epilogues bound, by their
// instructions and the latency of their few turns: 16,384 x 512 x 1,376 34 us, its gates 60 us, float32's of
// 18,500 x 97 x 250 30 us.
// float32 operands are sums of three bfloat16 planes (8 + 8 + 8 bits of mantissa), laid out by
// pack_kernel; a product of two is six products of planes, the three below 2^-24 left out.
#include <cuda_bf16.h>

#include "blackwell.cuh"

namespace rlenv {
namespace {

enum Activation { kSilu = 0, kGelu = 1 };

RLENV_D float reciprocal_approx(float x) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

// act(g) and act'(g): silu g / (1 + e^-g), or gelu g Phi(g) with the exact normal distribution. For bfloat16 results
// (half an ulp is 2^-9) the fast exponential and reciprocal are enough: __expf(x) is within 2 + 1.173 |x| ulp, 2^-20
// of its value where |x| < 5 and 2^-16 where it underflows, far out in silu's and gelu's negative tails. So is a
// polynomial for Phi: with z = |g| / sqrt 2 and t = 1 / (1 + 0.46 z), erfc(z) = e^(-z^2) t p(t), p of degree 7 fitted to
// erfc by least squares weighted towards the smallest largest relative error, 7.1e-7 with the coefficients as printed;
// e^(-z^2) serves the density too. The epilogue's instructions bound short contractions: gelu's gates of 16,384 x
// 512 x 1,376 take 68 us, with erfcf 97.
template <bool kFast, int kAct>
RLENV_D void activate(float g, float* y, float* slope) {
  if constexpr (kAct == kSilu) {
    const float s = kFast ? reciprocal_approx(1.0f + __expf(-g)) : 1.0f / (1.0f + expf(-g));
    *y = g * s;
    *slope = s * (1.0f + g * (1.0f - s));
  } else if constexpr (kFast) {
    const float t = reciprocal_approx(fmaf(0.325269119f, fabsf(g), 1.0f)), density = __expf(-0.5f * g * g);
    float p = 0.0338675529f;
    p = fmaf(p, t, -0.113352984f);
    p = fmaf(p, t, 0.0846521705f);
    p = fmaf(p, t, 0.0262626223f);
    p = fmaf(p, t, 0.0934411660f);
    p = fmaf(p, t, 0.115587331f);
    p = fmaf(p, t, 0.129778966f);
    p = fmaf(p, t, 0.129763514f);
    const float tail = density * t * p, cdf = g > 0.0f ? 1.0f - tail : tail;
    *y = g * cdf;
    *slope = fmaf(g * 0.39894228f, density, cdf);
  } else {
    const float cdf = 0.5f * erfcf(-0.70710678f * g);
    *y = g * cdf;
    *slope = cdf + g * (0.39894228f * expf(-0.5f * g * g));
  }
}

// ---- operands ------------------------------------------------------------------------------------

// The pitch of rows in scratch: whole lines of 128 bytes, so that a tensor copy's row of a tile lies in one
// (float32 4,330 x 881 x 1,780: 124 us against 184 with rows on 16 bytes, the gradient 502 against 698).
__host__ __device__ constexpr int64_t pitch_of(int64_t cols) { return (cols + 63) / 64 * 64; }

// Planes of up to three (rows, cols) arrays as bfloat16 (planes, rows, pitch_of(cols)): for
// float32 the three whose sum it is, for bfloat16 a copy (rows that are not on 16-byte boundaries). A warp takes
// a run of kPackRun columns of a row, a lane pairs of its elements. Bound by memory: 4,330 x 881 and twice 881 x
// 1,780 in float32, 69 MB, 10 us.
constexpr int kPackRun = 512;
struct Packing {
  const void* from[3];
  __nv_bfloat16* to[3];
  int64_t rows[3], cols[3], runs[4];  // runs: running
};
template <typename T, int kPlanes>
__global__ void __launch_bounds__(256) pack_kernel(const __grid_constant__ Packing p) {
  const int64_t i = int64_t(blockIdx.x) * 8 + (threadIdx.x >> 5);
  if (i >= p.runs[3]) return;
  const int a = i < p.runs[1] ? 0 : i < p.runs[2] ? 1 : 2;
  const int64_t rows = p.rows[a], cols = p.cols[a], pitch = pitch_of(cols);
  const uint32_t a_row = uint32_t((cols + kPackRun - 1) / kPackRun);
  const int64_t run = i - p.runs[a], r = a_row == 1 ? run : run / a_row, c0 = a_row == 1 ? 0 : run % a_row * kPackRun;
  const T* from = static_cast<const T*>(p.from[a]) + r * cols;
  __nv_bfloat16* to = p.to[a] + r * pitch;
  const int64_t first = c0 + 2 * (threadIdx.x & 31);
  const auto store = [&](int64_t c, float lo, float hi) {
#pragma unroll
    for (int q = 0; q < kPlanes; ++q) {
      const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
      *reinterpret_cast<__nv_bfloat162*>(to + q * rows * pitch + c) = v;
      lo -= __low2float(v), hi -= __high2float(v);
    }
  };
  constexpr int kAhead = kPlanes > 1 ? 8 : 4;  // pairs a lane loads before it stores any
#pragma unroll
  for (int u0 = 0; u0 < kPackRun / 64; u0 += kAhead) {
    if (c0 + 64 * u0 >= cols) break;
    float lo[kAhead], hi[kAhead];
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const int64_t c = first + 64 * (u0 + u);
      lo[u] = c < cols ? float(__ldg(from + c)) : 0.0f, hi[u] = c + 1 < cols ? float(__ldg(from + c + 1)) : 0.0f;
    }
#pragma unroll
    for (int u = 0; u < kAhead; ++u)
      if (first + 64 * (u0 + u) < cols) store(first + 64 * (u0 + u), lo[u], hi[u]);
  }
}

// ---- the product kernel ---------------------------------------------------------------------------

enum Op { kForward, kGates, kGradients };  // h; dg and du; dx, dWg and dWu

constexpr int kRows = 128;       // of a tile, in each block of a pair
constexpr int kBlock = 64;       // of the contraction: a tile row's 128 bytes
constexpr int kTmemColumns = 512, kBufferColumns = 256;
constexpr int kStageFloats = 32 * 32;  // the epilogue's tile of a warp

template <typename T, int kOp = kForward>
struct Tile {
  static constexpr bool kFloat = sizeof(T) == 4;
  static constexpr int kPlanes = kFloat ? 3 : 1;
  static constexpr int kCols = kFloat ? 128 : 256;
  static constexpr int kHalf = kCols / 2;        // columns of B in each block
  // Warps: copies, products, two idle ones, and those of the epilogue: sixteen where it computes (16,384 x 512 x
  // 1,376 in bfloat16, 34 us forward against 41 with eight, the gates 60 against 70). bfloat16's plain results want
  // the shared memory of the other eight as a sixth ring buffer (8,192 x 1,024 x 2,720, 125 us against 131).
  static constexpr int kEpilogue = kFloat || kOp != kGradients ? 16 : 8;
  static constexpr int kThreads = 128 + 32 * kEpilogue;
  static constexpr int kMine = kCols / (kEpilogue / 4);  // columns of the accumulator that a thread reads
  static constexpr int kStep = kBlock;
  static constexpr int kABytes = kRows * kBlock * 2;
  static constexpr int kRingBytes = kABytes + kHalf * kBlock * 2;  // a ring buffer: a plane of both operands
  static constexpr int kStages = kFloat || kOp == kGradients ? 6 : 5;
  static constexpr int kStageAt = kStages * kRingBytes;  // the epilogue's 32 x 32 tiles, one a warp
  // the ring starts on a 1,024-byte boundary
  static constexpr int kSmem = kStageAt + kEpilogue * kStageFloats * 4 + 1024;
  // Steps of the contraction summed in tensor memory before the epilogue takes them out into registers
  // (float32 only). The tensor core truncates as it accumulates; rounded additions of short sums keep
  // float32 results at float32's error. The leading planes' product and the five small ones have an
  // accumulator each: what is truncated of the small sums is small.
  static constexpr int kRun = 4;
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
  int splits, split_steps;   // of the contraction over tokens in the weights' gradients
  int dx_splits, dx_split_steps;  // of that over F in dx
  int extra;                      // rounds of dx's tiles for the pairs with fewer of the weights'
  const void* dh;            // kGates
  void *out, *dwg, *dwu;     // h or dx; the weights' gradients
  float *parts, *dx_parts;   // (splits, 2, K, F) where splits > 1, (dx_splits, M, K) where dx_splits > 1
  __nv_bfloat16* gates;      // (plane, dg or du, M, pitch)
  int64_t pitch;
  bool wide;                 // rows of h and dh start on the boundaries of fours
  bool turned;               // the weights' gradients are formed as their transposes, dg' x and du' x
};

// What pair `pair` of SMs works on, one item after the other: its share of the weights' tiles, then of dx's. The
// pairs with one of the weights' tiles fewer take kGradients' first `extra` rounds of dx's among themselves, and
// come first in the others.
struct Turn {
  int pairs, items, weights, mine, light, order, extra, at;
  RLENV_D Turn(const Product& p, int items, bool gradients) : items(items), at(0) {
    const int pair = blockIdx.x / 2;
    pairs = gridDim.x / 2;
    weights = gradients ? p.weight_rows * p.weight_cols * p.splits : 0;
    const int heavy = weights % pairs;  // pairs with a tile of the weights more
    mine = weights / pairs + (pair < heavy), light = pairs - heavy;
    order = pair < heavy ? light + pair : pair - heavy;
    extra = gradients ? p.extra : 0;
  }
  RLENV_D int next() {  // an item, or -1 after the last
    const int turn = at++, round = turn - mine;
    if (round < 0) return (order < light ? order + pairs - light : order - light) + turn * pairs;
    const bool early = order < light && round < extra;
    const int item = weights + (early ? round * light : extra * light + (order < light ? round - extra : round) * pairs) + order;
    return item < items ? item : -1;
  }
};

// Tiles are taken in bands of kBand rows of tiles, column by column, so that those in flight share
// operands that lie in L2.
constexpr int kBand = 8;

// A tile of work: columns from c0, rows from row tile `row`, a contraction over `steps` ring buffers of each of
// `segs` segments from the one numbered k0.
struct Work {
  bool weights;
  int weight, split, row, c0, k0, steps, segs;
};
template <typename T, int kOp>
RLENV_D Work work_of(const Product& p, int item) {
  constexpr int kStep = Tile<T>::kStep;
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
      w.k0 = w.split * p.split_steps;
      w.steps = min(p.split_steps, int((p.m + kStep - 1) / kStep) - w.k0);
    } else {
      item -= per * p.splits;
      const int tiles = rows * cols;
      w.split = item / tiles, item %= tiles;
      w.k0 = w.split * p.dx_split_steps;
      w.segs = 2, w.steps = min(p.dx_split_steps, int((p.f + kStep - 1) / kStep) - w.k0);
    }
  } else {
    w.steps = int((p.k + kStep - 1) / kStep);
  }
  const int per = kBand * cols, band = item / per, in = item % per;
  const int high = min(kBand, rows - band * kBand);
  w.row = band * kBand + in % high;
  int col = in / high;
  if (w.weights && col >= cols / 2) w.weight = 1, col -= cols / 2;
  w.c0 = col * (kOp == kGradients ? Tile<T>::kCols : Tile<T>::kHalf);
  return w;
}

// A step's planes in the order in which they are copied. A plane's products with those before it follow its
// arrival: 1 1, then 0 1, 1 0 and 0 0, then 0 2 and 2 0. Each is read from L2 once for all of its products
// (48 bytes a clock and SM; with a pass over the contraction for each product it was 96, more than L2 gives, and
// 4,330 x 881 x 1,780 forward took 125 us instead of 104), and the first buffer is free again halfway through.
template <typename T>
RLENV_D int plane_of(int turn) { return Tile<T>::kFloat ? 0x21 >> (2 * turn) & 3 : 0; }

// Four neighbouring values of a row, the first n of them there: in one access where all are and `wide`
// says that rows start on the boundaries of fours.
RLENV_D void store_four(float* to, float4 v, bool wide, int n) {
  if (wide && n >= 4) {
    *reinterpret_cast<float4*>(to) = v;
  } else {
    if (n > 0) to[0] = v.x;
    if (n > 1) to[1] = v.y;
    if (n > 2) to[2] = v.z;
    if (n > 3) to[3] = v.w;
  }
}
RLENV_D uint2 pack_four(float4 v) {
  const __nv_bfloat162 lo = __floats2bfloat162_rn(v.x, v.y), hi = __floats2bfloat162_rn(v.z, v.w);
  return make_uint2(*reinterpret_cast<const uint32_t*>(&lo), *reinterpret_cast<const uint32_t*>(&hi));
}
RLENV_D float4 unpack_four(uint2 w) {
  return make_float4(__uint_as_float(w.x << 16), __uint_as_float(w.x & 0xffff0000u), __uint_as_float(w.y << 16),
                     __uint_as_float(w.y & 0xffff0000u));
}
RLENV_D float4 unpack_four(float4 w) { return w; }
RLENV_D void store_four(__nv_bfloat16* to, float4 v, bool wide, int n) {
  if (wide && n >= 4) {
    *reinterpret_cast<uint2*>(to) = pack_four(v);
  } else {
    if (n > 0) to[0] = __float2bfloat16_rn(v.x);
    if (n > 1) to[1] = __float2bfloat16_rn(v.y);
    if (n > 2) to[2] = __float2bfloat16_rn(v.z);
    if (n > 3) to[3] = __float2bfloat16_rn(v.w);
  }
}
RLENV_D void load_four(const float* from, float4* v, bool wide, int n) {
  if (wide && n >= 4)
    *v = __ldg(reinterpret_cast<const float4*>(from));
  else
    *v = make_float4(n > 0 ? from[0] : 0.0f, n > 1 ? from[1] : 0.0f, n > 2 ? from[2] : 0.0f, n > 3 ? from[3] : 0.0f);
}
RLENV_D void load_four(const __nv_bfloat16* from, uint2* v, bool wide, int n) {
  if (wide && n >= 4) {
    *v = __ldg(reinterpret_cast<const uint2*>(from));
  } else {
    const unsigned short* f = reinterpret_cast<const unsigned short*>(from);
    *v = make_uint2((n > 0 ? f[0] : 0u) | (n > 1 ? uint32_t(f[1]) << 16 : 0u),
                    (n > 2 ? f[2] : 0u) | (n > 3 ? uint32_t(f[3]) << 16 : 0u));
  }
}
template <typename T>
struct Four {
  using type = float4;
};
template <>
struct Four<__nv_bfloat16> {
  using type = uint2;
};

// A warp's 32 x 32 tile of results goes through shared memory, written a row a lane and read four
// neighbours a lane, so that global accesses run along rows. Fours of columns are exchanged by the row's
// low three bits, which keeps both sides free of bank conflicts.
RLENV_D float4* stage_at(float* stage, int row, int four) {
  return reinterpret_cast<float4*>(stage) + row * 8 + (four ^ (row & 7));
}
// A gated tile is 16 columns of gates and their 16 ups: lane l has columns 4 (l % 4) .. + 3 of rows
// gated_row(l) + 8 i. Where the caller's rows do not start on the boundaries of fours, its values pass through
// the tile once more, so that a row's accesses are neighbours still: column l % 16 of rows lone_row(l, i).
RLENV_D int gated_row(int lane) { return (lane >> 2 & 1) * 4 + (lane >> 3); }
RLENV_D int lone_row(int lane, int i) { return (lane >> 4) * 4 + (i & 3) + (i >> 2) * 8; }
RLENV_D float& stage_one(float* stage, int row, int col) {
  return reinterpret_cast<float*>(stage_at(stage, row, col >> 2))[col & 3];
}

// The gradient dh of a gated tile, in a lane's order.
template <typename T>
RLENV_D void load_gradient(const Product& p, int64_t r0, int64_t c, typename Four<T>::type (&d)[4]) {
  const int lane = threadIdx.x & 31;
  const T* dh = static_cast<const T*>(p.dh) + r0 * p.f + c;
  const int rows = int(min(int64_t(32), p.m - r0)), cols = int(min(int64_t(16), p.f - c));
  if (p.wide) {
    const int col = lane % 4 * 4;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int r = gated_row(lane) + 8 * i;
      load_four(dh + r * p.f + col, &d[i], true, r < rows ? cols - col : 0);
    }
  } else {
    const int col = lane % 16;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      T v[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int r = lone_row(lane, 4 * i + j);
        v[j] = r < rows && col < cols ? dh[r * p.f + col] : T(0.0f);
      }
      if constexpr (sizeof(T) == 4) {
        d[i] = make_float4(v[0], v[1], v[2], v[3]);
      } else {
        const __nv_bfloat162 lo = __halves2bfloat162(v[0], v[1]), hi = __halves2bfloat162(v[2], v[3]);
        d[i] = make_uint2(*reinterpret_cast<const uint32_t*>(&lo), *reinterpret_cast<const uint32_t*>(&hi));
      }
    }
  }
}

template <typename T, int kOp, int kAct>
RLENV_D void finish_gated(const Product& p, int64_t r0, int64_t c, const typename Four<T>::type (&dh)[4], float* stage) {
  constexpr bool kFast = !Tile<T>::kFloat;
  const int lane = threadIdx.x & 31, col = lane % 4 * 4, lone = lane % 16;
  const int rows = int(min(int64_t(32), p.m - r0)), cols = int(min(int64_t(16), p.f - c));
  const int64_t plane = p.m * p.pitch;
  float4 g[4], u[4], d[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    g[i] = *stage_at(stage, gated_row(lane) + 8 * i, lane % 4);
    u[i] = *stage_at(stage, gated_row(lane) + 8 * i, 4 + lane % 4);
    if constexpr (kOp == kGates) d[i] = unpack_four(dh[i]);
  }
  if (kOp == kGates && !p.wide) {
    __syncwarp();
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      stage_one(stage, lone_row(lane, 4 * i), lone) = d[i].x;
      stage_one(stage, lone_row(lane, 4 * i + 1), lone) = d[i].y;
      stage_one(stage, lone_row(lane, 4 * i + 2), lone) = d[i].z;
      stage_one(stage, lone_row(lane, 4 * i + 3), lone) = d[i].w;
    }
    __syncwarp();
#pragma unroll
    for (int i = 0; i < 4; ++i) d[i] = *stage_at(stage, gated_row(lane) + 8 * i, lane % 4);
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int r = gated_row(lane) + 8 * i;
    float4 y, slope;
    activate<kFast, kAct>(g[i].x, &y.x, &slope.x);
    activate<kFast, kAct>(g[i].y, &y.y, &slope.y);
    activate<kFast, kAct>(g[i].z, &y.z, &slope.z);
    activate<kFast, kAct>(g[i].w, &y.w, &slope.w);
    if constexpr (kOp == kForward) {
      g[i] = make_float4(y.x * u[i].x, y.y * u[i].y, y.z * u[i].z, y.w * u[i].w);
      if (p.wide && r < rows) store_four(static_cast<T*>(p.out) + (r0 + r) * p.f + c + col, g[i], true, cols - col);
    } else if (r < rows && col < cols) {
      float4 dg = make_float4(d[i].x * u[i].x * slope.x, d[i].y * u[i].y * slope.y, d[i].z * u[i].z * slope.z,
                              d[i].w * u[i].w * slope.w);
      float4 du = make_float4(d[i].x * y.x, d[i].y * y.y, d[i].z * y.z, d[i].w * y.w);
      __nv_bfloat16* to = p.gates + (r0 + r) * p.pitch + c + col;  // the pitch holds whole eights
#pragma unroll
      for (int q = 0; q < Tile<T>::kPlanes; ++q, to += 2 * plane) {
        const uint2 a = pack_four(dg), b = pack_four(du);
        *reinterpret_cast<uint2*>(to) = a;
        *reinterpret_cast<uint2*>(to + plane) = b;
        const float4 x = unpack_four(a), z = unpack_four(b);
        dg.x -= x.x, dg.y -= x.y, dg.z -= x.z, dg.w -= x.w, du.x -= z.x, du.y -= z.y, du.z -= z.z, du.w -= z.w;
      }
    }
  }
  if (kOp == kForward && !p.wide) {
    __syncwarp();
#pragma unroll
    for (int i = 0; i < 4; ++i) *stage_at(stage, gated_row(lane) + 8 * i, lane % 4) = g[i];
    __syncwarp();
    T* const out = static_cast<T*>(p.out) + r0 * p.f + c + lone;
#pragma unroll 8
    for (int i = 0; i < 16; ++i) {
      const int r = lone_row(lane, i);
      if (r < rows && lone < cols) out[r * p.f] = T(stage_one(stage, r, lone));
    }
  }
}
template <typename T>
RLENV_D void finish_values(T* to, int64_t pitch, int64_t rows, int64_t cols, float* stage) {
  const int lane = threadIdx.x & 31;
  if (pitch % 4 == 0) {
    const int col = lane % 8 * 4, n = int(min(int64_t(4), cols - col));
    if (n <= 0) return;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int r = lane / 8 + 4 * i;
      if (r >= rows) return;
      store_four(to + r * pitch + col, *stage_at(stage, r, lane % 8), true, n);
    }
  } else if (lane < cols) {
#pragma unroll 8
    for (int r = 0; r < 32; ++r) {
      if (r >= rows) return;
      to[r * pitch + lane] = T(stage_one(stage, r, lane));
    }
  }
}

// Rows from r0, columns from c (of h, a weight or dx). v, as bits: 16 gates and 16 ups, or 32 values.
template <typename T, int kOp>
RLENV_D void finish(const Product& p, const Work& w, int64_t r0, int64_t c, const uint32_t (&v)[32],
                    const typename Four<T>::type (&dh)[4], float* stage) {
  const bool turned = kOp == kGradients && w.weights && p.turned;
  const int64_t all_rows = kOp != kGradients || !w.weights ? p.m : turned ? p.f : p.k;
  const int64_t all_cols = kOp == kGradients && (turned || !w.weights) ? p.k : p.f;
  if (r0 >= all_rows || c >= all_cols) return;
  const int lane = threadIdx.x & 31;
  if constexpr (kOp == kGradients && Tile<T>::kFloat) {
    if (turned) {  // a column of the tile lies in a row of the gradient
      float* to = p.splits > 1 ? p.parts + (int64_t(w.split) * 2 + w.weight) * p.k * p.f
                               : static_cast<float*>(w.weight ? p.dwu : p.dwg);
      to += c * p.f + r0 + lane;
      const int cols = int(min(int64_t(32), p.k - c));
      if (r0 + lane < p.f) {
#pragma unroll
        for (int i = 0; i < 32; ++i)
          if (i < cols) to[i * p.f] = __uint_as_float(v[i]);
      }
      return;
    }
  }
  __syncwarp();
#pragma unroll
  for (int i = 0; i < 8; ++i)
    *reinterpret_cast<uint4*>(stage_at(stage, lane, i)) = make_uint4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]);
  __syncwarp();
  if constexpr (kOp == kGradients) {
    if (w.weights && p.splits > 1)
      finish_values(p.parts + ((int64_t(w.split) * 2 + w.weight) * p.k + r0) * p.f + c, p.f, all_rows - r0,
                    all_cols - c, stage);
    else if (!w.weights && p.dx_splits > 1)
      finish_values(p.dx_parts + (int64_t(w.split) * p.m + r0) * p.k + c, p.k, all_rows - r0, all_cols - c, stage);
    else
      finish_values(static_cast<T*>(w.weights ? (w.weight ? p.dwu : p.dwg) : p.out) + r0 * all_cols + c, all_cols,
                    all_rows - r0, all_cols - c, stage);
  } else if (p.act == kSilu) {
    finish_gated<T, kOp, kSilu>(p, r0, c, dh, stage);
  } else {
    finish_gated<T, kOp, kGelu>(p, r0, c, dh, stage);
  }
}

template <typename T, int kOp>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(Tile<T, kOp>::kThreads, 1)
product_kernel(const __grid_constant__ Product p, int items) {
  using C = Tile<T, kOp>;
  constexpr bool kPaired = kOp != kGradients;  // half of a tile's columns are gates, half ups
  constexpr uint32_t kBox = 64 * kBlock * 2;
  extern __shared__ unsigned char raw[];
  __shared__ __align__(8) uint64_t bars[2 * C::kStages + 5];
  __shared__ uint32_t tmem_slot;
  __shared__ int dead_flag;
  __shared__ bw::Ending endings[2];  // of the pair's first block, and of its second
  volatile int* const dead = &dead_flag;
  const uint32_t ring = (bw::shared_at(raw) + 1023) & ~1023u;
  const uint32_t full = bw::shared_at(bars), empty = full + 8 * C::kStages;
  const uint32_t summed = empty + 8 * C::kStages, taken = summed + 16, drained = taken + 16;
  const int warp = __shfl_sync(0xffffffffu, int(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;
  const int rank = int(bw::cluster_rank());
  if (threadIdx.x == 0) {
    for (int i = 0; i < C::kStages; ++i) bw::barrier_init(full + 8 * i, 1), bw::barrier_init(empty + 8 * i, 1);
    for (int i = 0; i < 2; ++i) bw::barrier_init(summed + 8 * i, 1), bw::barrier_init(taken + 8 * i, 2 * C::kEpilogue);
    bw::barrier_init(drained, 1);
    dead_flag = 0, endings[rank] = bw::Ending{};
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 2) bw::tmem_alloc<kTmemColumns>(bw::shared_at(&tmem_slot));
  bw::fence_before();
  __syncthreads();
  bw::cluster_sync();
  bw::fence_after();
  const uint32_t tmem = __shfl_sync(0xffffffffu, tmem_slot, 0);
  Turn turns(p, items, kOp == kGradients);

  if (warp == 0) {
    // Both blocks copy their rows of A and their columns of B; all bytes count at the first block's barrier.
    int stage = 0, filled = 0;
    uint32_t phase = 0;
    bool ok = true;
    const uint32_t full_at = bw::in_block(full, 0);
    for (int item = turns.next(); item >= 0 && ok; item = turns.next()) {
      const Work w = work_of<T, kOp>(p, item);
      const Operands& in = p.in[kOp == kGradients && w.weights];
      const int r0 = (2 * w.row + rank) * kRows, c0 = w.c0 + (kPaired ? 0 : rank * C::kHalf);
      const CUtensorMap* const map_a = &in.a;
      for (int seg = 0; seg < w.segs && ok; ++seg) {
        // slices: planes; of the gates dg's and du's by turns. Gates in the first block, ups in the second.
        const CUtensorMap* const map_b = (kPaired ? rank : seg) ? &in.b1 : &in.b0;
        const int k_end = (w.k0 + w.steps) * C::kStep;
        for (int k = w.k0 * C::kStep; k < k_end && ok; k += C::kStep) {  // what lies past the contraction reads as zero
          for (int turn = 0; turn < C::kPlanes; ++turn) {
            const int plane = plane_of<T>(turn);
            const int of_gates = 2 * plane + (!kPaired && w.weights ? w.weight : seg);
            const int slice_a = !kPaired && (!w.weights || p.turned) ? of_gates : plane;
            const int slice_b = !kPaired && w.weights && !p.turned ? of_gates : plane;
            const uint32_t bar = full_at + 8 * stage, a = ring + stage * C::kRingBytes, b = a + C::kABytes;
            if (!(ok = bw::barrier_wait_warp(empty + 8 * stage, phase ^ 1, dead))) break;
            if (bw::elect()) {
              if (rank == 0) bw::barrier_expect(full + 8 * stage, 2 * C::kRingBytes);
              if (!kPaired && w.weights) {
#pragma unroll
                for (int i = 0; i < kRows / 64; ++i) bw::copy_tile(a + i * kBox, map_a, bar, r0 + 64 * i, k, slice_a);
              } else {
                bw::copy_tile(a, map_a, bar, k, r0, slice_a);
              }
              if (kPaired || w.weights) {
#pragma unroll
                for (int i = 0; i < C::kHalf / 64; ++i) bw::copy_tile(b + i * kBox, map_b, bar, c0 + 64 * i, k, slice_b);
              } else {
                bw::copy_tile(b, map_b, bar, k, c0, slice_b);
              }
            }
            ++filled;
            if (++stage == C::kStages) stage = 0, phase ^= 1;
          }
        }
      }
    }
    // Both blocks' buffers are released by the first block's commits: each block waits for the last release of every
    // buffer, so that no arrival is on its way to a block that has ended. (A release's parity is its round's.)
    for (int i = 0; i < C::kStages && ok; ++i)
      if (i < filled) ok = bw::barrier_wait_warp(empty + 8 * i, i < stage ? phase : phase ^ 1, dead);
    if (lane == 0) endings[rank].filled = filled;
  } else if (warp == 1) {
    if (rank == 0) {
      int stage = 0, buffer = 0, released = 0, runs = 0;
      uint32_t phase = 0, buffer_phase = 0;
      bool ok = true;
      for (int item = turns.next(); item >= 0 && ok; item = turns.next()) {
        const Work w = work_of<T, kOp>(p, item);
        const int steps = w.segs * w.steps;
        const bool mn_a = w.weights, mn_b = kPaired || w.weights;
        const uint32_t kind = bw::product_kind(2 * kRows, C::kCols, mn_a, mn_b);
        const uint32_t a0 = bw::operand(ring, mn_a, kBox), b0 = bw::operand(ring + C::kABytes, mn_b, kBox);
        const uint32_t a_step = mn_a ? 2048 / 16 : 32 / 16, b_step = mn_b ? 2048 / 16 : 32 / 16;  // 16 of the contraction
        int left = C::kFloat ? min(C::kRun, steps) : steps;  // steps to the end of the run
        bool more = false;                                   // the run has begun
        for (int it = 0; it < steps; ++it) {
          if (!more && !(ok = bw::barrier_wait_warp(taken + 8 * buffer, buffer_phase ^ 1, dead))) break;
          const uint32_t d = tmem + buffer * kBufferColumns, a = a0 + stage * (C::kRingBytes / 16),
                         b = b0 + stage * (C::kRingBytes / 16);
          const auto add = [&](uint32_t to, int of_a, int of_b, bool accumulate) {
#pragma unroll
            for (int k = 0; k < kBlock / 16; ++k)
              bw::multiply(to, a + of_a * (C::kRingBytes / 16) + k * a_step, b + of_b * (C::kRingBytes / 16) + k * b_step,
                           kind, k > 0 || accumulate);
          };
          const bool last = --left == 0;
#pragma unroll
          for (int turn = 0; turn < C::kPlanes; ++turn) {
            if (!(ok = bw::barrier_wait_warp(full + 8 * (stage + turn), phase, dead))) break;
            bw::fence_after();
            if (bw::elect()) {
              if (!C::kFloat) {
                add(d, 0, 0, more);
                bw::commit(empty + 8 * stage);
              } else if (turn == 0) {
                add(d + C::kCols, 0, 0, more);
              } else if (turn == 1) {
                add(d + C::kCols, 1, 0, true);
                add(d + C::kCols, 0, 1, true);
                bw::commit(empty + 8 * stage);
                add(d, 1, 1, more);
              } else {
                add(d + C::kCols, 1, 2, true);
                add(d + C::kCols, 2, 1, true);
                bw::commit(empty + 8 * (stage + 1));
                bw::commit(empty + 8 * (stage + 2));
              }
              if (last && turn == C::kPlanes - 1) bw::commit(summed + 8 * buffer);
            }
            released += C::kFloat ? turn : 1;  // none, one and two of a step's three
          }
          if (!ok) break;
          runs += last;
          more = !last;
          if (last) {
            if (++buffer == 2) buffer = 0, buffer_phase ^= 1;
            left = min(C::kRun, steps - it - 1);
          }
          if ((stage += C::kPlanes) == C::kStages) stage = 0, phase ^= 1;
        }
      }
      if (lane == 0) endings[0].released = released, endings[0].runs = runs;
    }
  } else if (warp >= 4) {
    const int quarter = warp & 3, part = (warp - 4) >> 2;
    float* const own_stage = reinterpret_cast<float*>(raw + (ring - bw::shared_at(raw)) + C::kStageAt) +
                             (warp - 4) * kStageFloats;
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
    // Run j of 32 columns of this thread's, as two of 16: a gated tile's are gates and ups.
    const auto column = [&](int j) { return kPaired ? part * (C::kMine / 2) + 16 * j : part * C::kMine + 32 * j; };
    constexpr int kRuns = C::kMine / 32;
    const auto load_run = [&](uint32_t (&v)[32], int j, int from = 0) {
      const uint32_t at = tmem + lanes + buffer * kBufferColumns + from + column(j);
      bw::tmem_load16x2(v, at, at + (kPaired ? C::kHalf : 16));
    };
    // A run of results goes out while the next one's accumulators and gradients are on their way, the next tile's
    // first gradients among them.
    typename Four<T>::type dh[2][4];
    const auto rows_of = [&](const Work& w) { return int64_t(2 * w.row + rank) * kRows + 32 * quarter; };
    int item = turns.next();
    Work next = item >= 0 ? work_of<T, kOp>(p, item) : Work{};
    const auto load_dh = [&](const Work& w, int j) {
      if constexpr (kOp == kGates) load_gradient<T>(p, rows_of(w), w.c0 + column(j), dh[j & 1]);
    };
    if (item >= 0) load_dh(next, 0);
    while (item >= 0) {
      const Work w = next;
      item = turns.next();
      const bool another = item >= 0;
      if (another) next = work_of<T, kOp>(p, item);
      const int64_t r0 = rows_of(w);
      const auto finish_run = [&](uint32_t (&v)[32], int j, const typename Four<T>::type (&d)[4]) {
        if (!ok) {  // a wait ran out: the results say so
#pragma unroll
          for (int i = 0; i < 32; ++i) v[i] = 0x7fffffffu;
        }
        finish<T, kOp>(p, w, r0, w.c0 + column(j), v, d, own_stage);
        __syncwarp();  // lanes part over rows and columns that are not there; what follows is the whole warp's
      };
      if constexpr (C::kFloat) {
        float sum[kRuns][32];
#pragma unroll
        for (int j = 0; j < kRuns; ++j)
#pragma unroll
          for (int i = 0; i < 32; ++i) sum[j][i] = 0.0f;
        for (int left = w.segs * w.steps; left > 0; left -= C::kRun) {
          if (!(ok = ok && bw::barrier_wait_warp(summed + 8 * buffer, buffer_phase, dead))) break;
          bw::fence_after();
#pragma unroll
          for (int j = 0; j < kRuns; ++j)
#pragma unroll
            for (int from = 0; from <= C::kCols; from += C::kCols) {
              uint32_t v[32];
              load_run(v, j, from);
              bw::tmem_ready(v);
#pragma unroll
              for (int i = 0; i < 32; ++i) sum[j][i] += __uint_as_float(v[i]);
            }
          take_next();
        }
        static_assert(kRuns == 1, "a float32 tile's columns are one run a thread");
        uint32_t v[32];
#pragma unroll
        for (int i = 0; i < 32; ++i) v[i] = __float_as_uint(sum[0][i]);
        typename Four<T>::type d[4] = {dh[0][0], dh[0][1], dh[0][2], dh[0][3]};
        if (another) load_dh(next, 0);
        finish_run(v, 0, d);
      } else {
        ok = ok && bw::barrier_wait_warp(summed + 8 * buffer, buffer_phase, dead);
        bw::fence_after();
        // Where the registers allow, the next run is read while this one goes out.
        constexpr int kAhead = kOp == kGradients;
        uint32_t v[1 + kAhead][32];
        load_run(v[0], 0);
#pragma unroll
        for (int j = 0; j < kRuns; ++j) {
          bw::tmem_ready(v[j & kAhead]);
          if (kAhead && j + 1 < kRuns) load_run(v[(j + 1) & kAhead], j + 1);
          if (ok && j + 1 == kRuns) take_next();  // all of the accumulator is read
          if (j + 1 < kRuns) load_dh(w, j + 1);
          else if (another) load_dh(next, 0);
          finish_run(v[j & kAhead], j, dh[j & 1]);
          if (!kAhead && j + 1 < kRuns) load_run(v[0], j + 1);
        }
      }
    }
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
  if (warp == 2) bw::tmem_free<kTmemColumns>(tmem);
}

// The gradients from the sums over parts of their contractions: both weights' from `splits` parts of tokens,
// dx's from `dx_splits` parts of F (0: it is whole already).
template <typename T>
__global__ void __launch_bounds__(256)
add_parts_kernel(const float* __restrict__ parts, int splits, int64_t size, T* __restrict__ dwg, T* __restrict__ dwu,
                 const float* __restrict__ dx_parts, int dx_splits, int64_t dx_size, T* __restrict__ dx) {
  int64_t e = int64_t(blockIdx.x) * 256 + threadIdx.x;
  const int64_t weights = splits > 1 ? 2 * size : 0;
  const bool of_dx = e >= weights;
  if (of_dx) e -= weights;
  if (of_dx && (dx_splits <= 1 || e >= dx_size)) return;
  const float* from = of_dx ? dx_parts : parts;
  const int64_t stride = of_dx ? dx_size : 2 * size;
  const int count = of_dx ? dx_splits : splits;
  float sum = 0.0f;
#pragma unroll 8
  for (int s = 0; s < count; ++s) sum += __ldg(from + s * stride + e);
  T* to = of_dx ? dx : e < size ? dwg : dwu;
  to[!of_dx && e >= size ? e - size : e] = T(sum);
}

// ---- few rows ----------------------------------------------------------------------------------------

// h for up to kFew rows of x at a time, a policy acting: matrix-vector products, bound by reading the
// weights (1,024 x 4,096 in bfloat16, one row: 5.1 us with the weights in L2, 3.3 TB/s; eight rows, 11.4 us, are
// bound by the products). A block owns 32 columns of both weights, so that 148 blocks read at once; its warps
// split the contraction, each thread reading 16 bytes of every kApart-th row, and the sums meet in shared memory
// in a fixed order. kGrad: with dh, the gates' gradients dg and du in float32, (2, m, pitch) with pitch f rounded
// up to four and zeros there.
constexpr int kFewThreads = 256, kFewCols = 32;

template <typename T, bool kWide>
RLENV_D void load_columns(const T* p, int n, float (&v)[16 / sizeof(T)]) {
  constexpr int kPer = 16 / sizeof(T);
  if constexpr (kWide && sizeof(T) == 2) {
    const uint4 w = __ldg(reinterpret_cast<const uint4*>(p));
    const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) v[2 * i] = __uint_as_float(u[i] << 16), v[2 * i + 1] = __uint_as_float(u[i] & 0xffff0000u);
  } else if constexpr (kWide) {
    const float4 w = __ldg(reinterpret_cast<const float4*>(p));
    v[0] = w.x, v[1] = w.y, v[2] = w.z, v[3] = w.w;
  } else {
#pragma unroll
    for (int i = 0; i < kPer; ++i) v[i] = i < n ? float(p[i]) : 0.0f;
  }
}

template <typename T, int kFew, bool kWide, bool kGrad>
__global__ void __launch_bounds__(kFewThreads)
few_rows_kernel(const T* __restrict__ x, const T* __restrict__ wg, const T* __restrict__ wu, int64_t m, int64_t k,
                int64_t f, int act, T* __restrict__ out, const T* __restrict__ dh, float* __restrict__ gates) {
  constexpr int kPer = 16 / sizeof(T), kAcross = kFewCols / kPer, kApart = kFewThreads / kAcross;
  constexpr int kUnroll = kFew > 4 ? 4 : 8;
  __shared__ float parts[kFewThreads / 32][2 * kFew * kFewCols];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, own = lane % kAcross * kPer;
  const int64_t c = int64_t(blockIdx.x) * kFewCols + own, m0 = int64_t(blockIdx.y) * kFew;
  const int n = int(min(int64_t(kPer), max(int64_t(0), f - c)));
  float g[kFew][kPer] = {}, u[kFew][kPer] = {};
  if (n > 0) {
#pragma unroll kUnroll
    for (int64_t i = threadIdx.x / kAcross; i < k; i += kApart) {
      float a[kPer], b[kPer];
      load_columns<T, kWide>(wg + i * f + c, n, a);
      load_columns<T, kWide>(wu + i * f + c, n, b);
#pragma unroll
      for (int r = 0; r < kFew; ++r) {
        const float xr = m0 + r < m ? float(x[(m0 + r) * k + i]) : 0.0f;
#pragma unroll
        for (int j = 0; j < kPer; ++j) g[r][j] = fmaf(xr, a[j], g[r][j]), u[r][j] = fmaf(xr, b[j], u[r][j]);
      }
    }
  }
#pragma unroll
  for (int r = 0; r < kFew; ++r)
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
#pragma unroll
      for (int o = 16; o >= kAcross; o >>= 1) {
        g[r][j] += __shfl_xor_sync(0xffffffffu, g[r][j], o);
        u[r][j] += __shfl_xor_sync(0xffffffffu, u[r][j], o);
      }
      if (lane < kAcross) {
        parts[warp][r * kFewCols + own + j] = g[r][j];
        parts[warp][(kFew + r) * kFewCols + own + j] = u[r][j];
      }
    }
  __syncthreads();
  for (int e = threadIdx.x; e < kFew * kFewCols; e += kFewThreads) {
    const int64_t r = m0 + e / kFewCols, col = int64_t(blockIdx.x) * kFewCols + e % kFewCols;
    const int64_t pitch = (f + 3) / 4 * 4;
    if (kGrad && r < m && col >= f && col < pitch) gates[r * pitch + col] = gates[(m + r) * pitch + col] = 0.0f;
    if (r >= m || col >= f) continue;
    float sg = 0.0f, su = 0.0f;
#pragma unroll
    for (int w = 0; w < kFewThreads / 32; ++w) sg += parts[w][e], su += parts[w][kFew * kFewCols + e];
    float y, slope;
    if (act == kSilu) activate<false, kSilu>(sg, &y, &slope);
    else activate<false, kGelu>(sg, &y, &slope);
    if constexpr (kGrad) {
      const float d = float(dh[r * f + col]);
      gates[r * pitch + col] = d * su * slope;
      gates[(m + r) * pitch + col] = d * y;
    } else {
      out[r * f + col] = T(y * su);
    }
  }
}

// Four neighbours of a row, those from n on as zeros and not written.
template <typename T, bool kWide>
RLENV_D float4 load_four(const T* p, int64_t n) {
  if constexpr (kWide && sizeof(T) == 2) {
    const uint2 w = __ldg(reinterpret_cast<const uint2*>(p));
    return make_float4(__uint_as_float(w.x << 16), __uint_as_float(w.x & 0xffff0000u), __uint_as_float(w.y << 16),
                       __uint_as_float(w.y & 0xffff0000u));
  } else if constexpr (kWide) {
    return __ldg(reinterpret_cast<const float4*>(p));
  } else {
    return make_float4(n > 0 ? float(p[0]) : 0.0f, n > 1 ? float(p[1]) : 0.0f, n > 2 ? float(p[2]) : 0.0f,
                       n > 3 ? float(p[3]) : 0.0f);
  }
}
template <typename T, bool kWide>
RLENV_D void store_four(T* p, const float (&v)[4], int64_t n) {
  if constexpr (kWide && sizeof(T) == 2) {
    const __nv_bfloat162 lo = __floats2bfloat162_rn(v[0], v[1]), hi = __floats2bfloat162_rn(v[2], v[3]);
    *reinterpret_cast<uint2*>(p) =
        make_uint2(*reinterpret_cast<const uint32_t*>(&lo), *reinterpret_cast<const uint32_t*>(&hi));
  } else if constexpr (kWide) {
    *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (i < n) p[i] = T(v[i]);
  }
}
RLENV_D float dot_four(const float4& a, const float4& b, float sum) {
  return fmaf(a.x, b.x, fmaf(a.y, b.y, fmaf(a.z, b.z, fmaf(a.w, b.w, sum))));
}

// The gradients of few rows from dg and du (`gates`, as above). Bound by writing both weights' gradients and
// reading the weights: a float32 row of 1,024 x 4,096 20 us with the gates' launch, 100 MB in all, 5 TB/s (in turns
// that find the weights in L2); from some eight rows on by the products. The first blocks form a 64 x 64 tile of
// both weights' gradients each, sums over the tokens in registers; the others dx of kFew tokens at four columns, dot
// products of whole rows of the weights, whose sums meet in shared memory in a fixed order.
constexpr int kFewTile = 64, kFewTokens = 8, kFewDx = 4;
struct FewGradients {
  const void *x, *wg, *wu;
  const float* gates;
  void *dx, *dwg, *dwu;
  int64_t m, k, f;
  uint32_t across, weight_blocks, dx_across;
};

template <typename T, int kFew, bool kWide>
__global__ void __launch_bounds__(kFewThreads) few_gradients_kernel(const FewGradients p) {
  const int64_t pitch = (p.f + 3) / 4 * 4;
  const float *const dg = p.gates, *const du = p.gates + p.m * pitch;
  if (blockIdx.x < p.weight_blocks) {
    __shared__ __align__(16) float d[2][kFewTokens][kFewTile], x[kFewTokens][kFewTile];
    const int64_t c0 = int64_t(blockIdx.x % p.across) * kFewTile, r0 = int64_t(blockIdx.x / p.across) * kFewTile;
    const int own_c = threadIdx.x % 16 * 4, own_r = threadIdx.x / 16 * 4;
    float g[4][4] = {}, u[4][4] = {};
    for (int64_t m0 = 0; m0 < p.m; m0 += kFewTokens) {
      const int which = threadIdx.x / 128, token = threadIdx.x / 16 % kFewTokens;
      *reinterpret_cast<float4*>(&d[which][token][own_c]) =
          m0 + token < p.m && c0 + own_c < pitch
              ? __ldg(reinterpret_cast<const float4*>((which ? du : dg) + (m0 + token) * pitch + c0 + own_c))
              : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      for (int e = threadIdx.x; e < kFewTokens * kFewTile; e += kFewThreads) {
        const int64_t t = m0 + e / kFewTile, r = r0 + e % kFewTile;
        x[e / kFewTile][e % kFewTile] = t < p.m && r < p.k ? float(static_cast<const T*>(p.x)[t * p.k + r]) : 0.0f;
      }
      __syncthreads();
#pragma unroll
      for (int t = 0; t < kFewTokens; ++t) {
        const float4 a = *reinterpret_cast<const float4*>(&x[t][own_r]);
        const float4 b = *reinterpret_cast<const float4*>(&d[0][t][own_c]);
        const float4 c = *reinterpret_cast<const float4*>(&d[1][t][own_c]);
        const float av[4] = {a.x, a.y, a.z, a.w}, bv[4] = {b.x, b.y, b.z, b.w}, cv[4] = {c.x, c.y, c.z, c.w};
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int j = 0; j < 4; ++j) g[i][j] = fmaf(av[i], bv[j], g[i][j]), u[i][j] = fmaf(av[i], cv[j], u[i][j]);
      }
      __syncthreads();
    }
    const int64_t c = c0 + own_c;
    if (c >= p.f) return;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int64_t r = r0 + own_r + i;
      if (r >= p.k) return;
      store_four<T, kWide>(static_cast<T*>(p.dwg) + r * p.f + c, g[i], p.f - c);
      store_four<T, kWide>(static_cast<T*>(p.dwu) + r * p.f + c, u[i], p.f - c);
    }
    return;
  }
  __shared__ float parts[kFewThreads / 32][kFewDx * kFew];
  const uint32_t id = blockIdx.x - p.weight_blocks;
  const int64_t k0 = int64_t(id % p.dx_across) * kFewDx, m0 = int64_t(id / p.dx_across) * kFew;
  float sum[kFewDx][kFew] = {};
  for (int64_t c = 4 * threadIdx.x; c < p.f; c += 4 * kFewThreads) {
    float4 g[kFewDx], u[kFewDx];
#pragma unroll
    for (int i = 0; i < kFewDx; ++i) {
      const int64_t at = (k0 + i < p.k ? k0 + i : p.k - 1) * p.f + c;
      g[i] = load_four<T, kWide>(static_cast<const T*>(p.wg) + at, p.f - c);
      u[i] = load_four<T, kWide>(static_cast<const T*>(p.wu) + at, p.f - c);
    }
#pragma unroll
    for (int t = 0; t < kFew; ++t) {
      const int64_t at = (m0 + t < p.m ? m0 + t : p.m - 1) * pitch + c;
      const float4 b = __ldg(reinterpret_cast<const float4*>(dg + at)), w = __ldg(reinterpret_cast<const float4*>(du + at));
#pragma unroll
      for (int i = 0; i < kFewDx; ++i) sum[i][t] = dot_four(u[i], w, dot_four(g[i], b, sum[i][t]));
    }
  }
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int i = 0; i < kFewDx; ++i)
#pragma unroll
    for (int t = 0; t < kFew; ++t) {
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) sum[i][t] += __shfl_xor_sync(0xffffffffu, sum[i][t], o);
      if (lane == 0) parts[warp][t * kFewDx + i] = sum[i][t];
    }
  __syncthreads();
  const int t = threadIdx.x / kFewDx, i = threadIdx.x % kFewDx;
  if (t >= kFew || m0 + t >= p.m || k0 + i >= p.k) return;
  float whole = 0.0f;
#pragma unroll
  for (int w = 0; w < kFewThreads / 32; ++w) whole += parts[w][threadIdx.x];
  static_cast<T*>(p.dx)[(m0 + t) * p.k + k0 + i] = T(whole);
}

template <typename T, int kFew>
int few_rows(const void* x, const void* wg, const void* wu, int64_t m, int64_t k, int64_t f, int act, void* out,
             const void* dh, void* gates, void* dx, void* dwg, void* dwu, cudaStream_t s) {
  const dim3 grid(unsigned((f + kFewCols - 1) / kFewCols), unsigned((m + kFew - 1) / kFew));
  const T *X = static_cast<const T*>(x), *G = static_cast<const T*>(wg), *U = static_cast<const T*>(wu);
  const T* const D = static_cast<const T*>(dh);
  T* const to = static_cast<T*>(out);
  float* const own = static_cast<float*>(gates);
  const bool wide = f * int64_t(sizeof(T)) % 16 == 0;
  if (!dh) {
    if (wide) few_rows_kernel<T, kFew, true, false><<<grid, kFewThreads, 0, s>>>(X, G, U, m, k, f, act, to, D, own);
    else few_rows_kernel<T, kFew, false, false><<<grid, kFewThreads, 0, s>>>(X, G, U, m, k, f, act, to, D, own);
    return launch_status();
  }
  FewGradients p{x, wg, wu, own, dx, dwg, dwu, m, k, f, 0, 0, 0};
  const int64_t across = (f + kFewTile - 1) / kFewTile, weight_blocks = across * ((k + kFewTile - 1) / kFewTile);
  const int64_t dx_across = (k + kFewDx - 1) / kFewDx, blocks = weight_blocks + dx_across * ((m + kFew - 1) / kFew);
  if (blocks > 0x7fffffff) return RLENV_EINVAL;
  p.across = uint32_t(across), p.weight_blocks = uint32_t(weight_blocks), p.dx_across = uint32_t(dx_across);
  if (wide) few_rows_kernel<T, kFew, true, true><<<grid, kFewThreads, 0, s>>>(X, G, U, m, k, f, act, to, D, own);
  else few_rows_kernel<T, kFew, false, true><<<grid, kFewThreads, 0, s>>>(X, G, U, m, k, f, act, to, D, own);
  if (const int rc = launch_status()) return rc;
  if (f % 4 == 0) few_gradients_kernel<T, kFew, true><<<unsigned(blocks), kFewThreads, 0, s>>>(p);
  else few_gradients_kernel<T, kFew, false><<<unsigned(blocks), kFewThreads, 0, s>>>(p);
  return launch_status();
}

// Whether the products are formed this way: a few rows in any case, more where the blocks of 8 rows and 32
// columns are one round on the SMs (bfloat16) or three (float32, whose tiles have the weights laid out as planes
// first). Measured in us, this way and by tiles: bfloat16 1,024 x 4,096, 1 row 5.0 and 12.9, 8 rows 11.3 and 10.7,
// 16 rows 21.0 and 10.6; 1,024 x 16,384, 4 rows 21.8 and 21.1, 8 rows 38.7 and 20.9; 512 x 512, 72 rows 8.0 and
// 8.3, 96 rows 14.6 and 8.4; 4,096 x 1,024, 16 rows 29.2 and 23.8 (the rule's worst); float32 1,024 x 4,096, 24
// rows 26.4 and 31.4, 32 rows 34.5 and 31.4; 1,024 x 16,384, 16 rows 108 and 125, 24 rows 165 and 121; 512 x 512,
// 192 rows 16.3 and 15.9, 256 rows 21.1 and 16.0; 97 x 250, 256 rows 7.5 and 10.7, 448 rows 13.4 and 10.9.
bool few_rows_fit(int dtype, int64_t m, int64_t f) {
  const bool wide = dtype == RLENV_F32;
  const int64_t blocks = (m + 7) / 8 * ((f + kFewCols - 1) / kFewCols);
  return m <= (wide ? 16 : 4) || blocks <= 148 * (wide ? 3 : 1);
}
// The same for the gradient, whose tiles cost a launch or two more and work on 256 rows however few there are; this
// way takes longer by the row. Measured in us, this way and by tiles: float32 1,024 x 4,096, 1 row 20 and 73, 16
// rows 53 and 67, 24 rows 73 and 67; 1,024 x 1,024, 32 rows 29.5 and 39.9, 48 rows 45 and 40; 83 x 3,683, 48 rows
// 28.1 and 29.6, 64 rows 35.6 and 29.7; 512 x 512, 64 rows 20 and 28. bfloat16 922 x 5,556, 4 rows 39 and 43, 8
// rows 52 and 40; 1,024 x 4,096, 8 rows 28.3 and 30.3; 97 x 250, 32 rows 14 and 20; 512 x 512, 8 rows 11 and 20, 32
// rows 16 and 21; 83 x 3,683, 16 rows 26 and 23; 2,000 x 100, 4 rows 24 and 25.5, 8 rows 32 and 25.5.
bool few_gradients_fit(int dtype, int64_t m, int64_t k, int64_t f) {
  const double products = double(m) * double(k) * double(f);
  return dtype == RLENV_F32 ? m <= 16 || (m <= 48 && products <= 33554432.0)
                            : m <= 4 || (m <= 32 && products <= 2097152.0);
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
  float *parts, *dx_parts;
  int splits, split_steps, dx_splits, dx_split_steps, extra;
  int64_t bytes;
};

constexpr int kPairsOfSms = 74;
constexpr int64_t kFewestSteps = 8;

// Whether the weights' gradients take fewer tiles as their transposes: a tile of float32 values is twice as high as
// wide (18,500 x 97 x 250: both gradients 29 us against 35).
bool turns(int dtype, int64_t k, int64_t f) {
  constexpr int64_t kHigh = 2 * kRows, kWide = Tile<float>::kCols;
  return dtype == RLENV_F32 && round_up(f, kHigh) * round_up(k, kWide) < round_up(k, kHigh) * round_up(f, kWide);
}

// The longest share of a pair of SMs, in steps, when the weights' tiles of Lw steps and dx's of Ld are dealt as
// Turn does, with `extra` rounds of dx's for the pairs that have a tile of the weights fewer.
double longest_share(int64_t weights, double lw, int64_t dx, double ld, int64_t extra) {
  const int64_t pairs = weights + dx < kPairsOfSms ? weights + dx : kPairsOfSms;
  const int64_t each = weights / pairs, heavy = weights % pairs, light = pairs - heavy;
  const int64_t rest = dx > extra * light ? dx - extra * light : 0, rounds = rest / pairs, left = rest % pairs;
  const double a = heavy ? (each + 1) * lw + (rounds + (left > light)) * ld : 0.0;
  const double b = each * lw + (extra + rounds + (left > 0)) * ld;
  return a > b ? a : b;
}

// The gradients' contractions are split where a tile would take longer than a pair of SMs' share of all the
// work, or the shares would be uneven: a small block's weights are a few tiles, each a sum over every token; few
// tokens' dx a few, each a sum over all of F. The parts' sums are kept in float32 and added up in order, which
// costs their writing and reading, at some 5 TB/s, and a launch, 4 us. Of the numbers of parts from the least
// that keeps a tile within the share to three more, the ones with the shortest longest share, plus that cost.
void split_gradients(int dtype, int64_t m, int64_t k, int64_t f, Layout* l) {
  const bool is_float = dtype == RLENV_F32;
  const int64_t wide = is_float ? Tile<float>::kCols : Tile<__nv_bfloat16>::kCols, high = 2 * kRows;
  const int64_t rows = turns(dtype, k, f) ? f : k, cols = turns(dtype, k, f) ? k : f;
  const int64_t steps = (m + kBlock - 1) / kBlock, tiles = (rows + high - 1) / high * ((cols + wide - 1) / wide) * 2;
  const int64_t dx_steps = (f + kBlock - 1) / kBlock, dx_tiles = (m + high - 1) / high * ((k + wide - 1) / wide);
  // A step's time; what a tile takes besides its steps, and at the least (its epilogue), in steps. As measured.
  const double step_us = is_float ? 1.06 : 0.36, turn = 0.5, least = is_float ? 2.0 : 10.0;
  const auto length = [&](int64_t n) { return turn + (n > least ? n : least); };
  int64_t share = (tiles * steps + 2 * dx_tiles * dx_steps) / kPairsOfSms;
  if (share < kFewestSteps) share = kFewestSteps;
  double best = 0.0;
  const int64_t a0 = (steps + share - 1) / share, b0 = (2 * dx_steps + share - 1) / share;
  for (int64_t i = 0; i < 4; ++i)
    for (int64_t j = 0; j < 4; ++j) {
      const int64_t each = (steps + a0 + i - 1) / (a0 + i), dx_each = (dx_steps + b0 + j - 1) / (b0 + j);
      const int64_t a = (steps + each - 1) / each, b = (dx_steps + dx_each - 1) / dx_each;
      const double bytes = (a > 1 ? 16.0 * a * k * f : 0.0) + (b > 1 ? 8.0 * b * m * k : 0.0);
      const double cost = bytes > 0.0 ? (4.0 + bytes / 5e6) / step_us : 0.0, lw = length(each), ld = length(2 * dx_each);
      for (int64_t extra = int64_t(lw / ld); extra <= int64_t(lw / ld) + 1; ++extra) {
        const double all = cost + longest_share(tiles * a, lw, dx_tiles * b, ld, extra);
        if (best > 0.0 && all >= best) continue;
        best = all;
        l->splits = int(a), l->split_steps = int(each), l->dx_splits = int(b), l->dx_split_steps = int(dx_each);
        l->extra = int(extra);
      }
    }
}
Layout lay_out(int dtype, int64_t m, int64_t k, int64_t f, bool backward, void* scratch) {
  Scratch s{static_cast<unsigned char*>(scratch), 0};
  Layout l{};
  const int64_t n = planes(dtype);
  if (!backward && few_rows_fit(dtype, m, f)) return l;
  if (backward && few_gradients_fit(dtype, m, k, f)) {
    l.gates = s.take(2 * m * round_up(f, 4) * 4);
    l.bytes = s.used;
    return l;
  }
  if (packs(dtype, k)) l.x = s.take(n * m * pitch_of(k) * 2);
  if (packs(dtype, f)) l.wg = s.take(n * k * pitch_of(f) * 2), l.wu = s.take(n * k * pitch_of(f) * 2);
  if (backward) {
    l.gates = s.take(2 * n * m * pitch_of(f) * 2);
    if (m > 0 && k > 0 && f > 0) split_gradients(dtype, m, k, f, &l);
    if (l.splits > 1) l.parts = static_cast<float*>(s.take(int64_t(l.splits) * 2 * k * f * 4));
    if (l.dx_splits > 1) l.dx_parts = static_cast<float*>(s.take(int64_t(l.dx_splits) * m * k * 4));
  }
  l.bytes = s.used;
  return l;
}

// The operands of the caller's arrays, the ones that need it packed in one launch.
template <typename T>
int operands(const void* const (&from)[3], const int64_t (&rows)[3], const int64_t (&cols)[3], void* const (&packed)[3],
             cudaStream_t s, Operand (&o)[3]) {
  constexpr int kPlanes = Tile<T>::kPlanes;
  Packing p{};
  for (int i = 0; i < 3; ++i) {
    p.runs[i + 1] = p.runs[i];
    if (!packed[i]) {
      o[i] = {static_cast<const __nv_bfloat16*>(from[i]), rows[i], cols[i], cols[i], 1};
      continue;
    }
    p.from[i] = from[i], p.to[i] = static_cast<__nv_bfloat16*>(packed[i]);
    p.rows[i] = rows[i], p.cols[i] = cols[i], p.runs[i + 1] += rows[i] * ((cols[i] + kPackRun - 1) / kPackRun);
    o[i] = {p.to[i], rows[i], cols[i], pitch_of(cols[i]), kPlanes};
  }
  if (p.runs[3] == 0) return RLENV_OK;
  if ((p.runs[3] + 7) / 8 > 0x7fffffff) return RLENV_EINVAL;
  pack_kernel<T, kPlanes><<<grid_for(p.runs[3], 8), 256, 0, s>>>(p);
  return launch_status();
}

template <typename T, int kOp>
int run_product(const Product& p, cudaStream_t s) {
  using C = Tile<T, kOp>;
  const int64_t items = int64_t(p.row_tiles) * p.col_tiles * (kOp == kGradients ? p.dx_splits : 1) +
                        int64_t(p.weight_rows) * p.weight_cols * p.splits;
  if (items > 0x7fff0000) return RLENV_EINVAL;
  int dev = 0, sms = 0;
  if (cudaError_t e = cudaGetDevice(&dev)) return int(e);
  if (cudaError_t e = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev)) return int(e);
  if (cudaError_t e = cudaFuncSetAttribute(product_kernel<T, kOp>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmem))
    return int(e);
  const int grid = 2 * int(items < sms / 2 ? items : sms / 2);
  product_kernel<T, kOp><<<grid, C::kThreads, C::kSmem, s>>>(p, int(items));
  return launch_status();
}

int tile_count(int64_t n, int64_t of) { return int((n + of - 1) / of); }

template <typename T>
int ffn(const void* dh, const void* x, const void* wg, const void* wu, int64_t m, int64_t k, int64_t f, int act,
        void* out, void* dx, void* dwg, void* dwu, const Layout& l, cudaStream_t s) {
  using C = Tile<T>;
  constexpr int kDtype = C::kFloat ? RLENV_F32 : RLENV_BF16;
  if (dh ? few_gradients_fit(kDtype, m, k, f) : few_rows_fit(kDtype, m, f))
    return m == 1   ? few_rows<T, 1>(x, wg, wu, m, k, f, act, out, dh, l.gates, dx, dwg, dwu, s)
           : m == 2 ? few_rows<T, 2>(x, wg, wu, m, k, f, act, out, dh, l.gates, dx, dwg, dwu, s)
           : m <= 4 ? few_rows<T, 4>(x, wg, wu, m, k, f, act, out, dh, l.gates, dx, dwg, dwu, s)
                    : few_rows<T, 8>(x, wg, wu, m, k, f, act, out, dh, l.gates, dx, dwg, dwu, s);
  Operand in[3];
  if (const int rc = operands<T>({x, wg, wu}, {m, k, k}, {k, f, f}, {l.x, l.wg, l.wu}, s, in)) return rc;
  const Operand &X = in[0], &G = in[1], &U = in[2];
  Product p{};
  p.m = m, p.k = k, p.f = f, p.act = act, p.out = out, p.dh = dh;
  p.gates = static_cast<__nv_bfloat16*>(l.gates), p.pitch = pitch_of(f);
  p.wide = f % 4 == 0 && reinterpret_cast<uintptr_t>(dh) % (4 * sizeof(T)) == 0;
  p.row_tiles = tile_count(m, 2 * kRows), p.col_tiles = tile_count(f, C::kHalf);
  if (const int rc = X.map(&p.in[0].a, kRows)) return rc;
  if (const int rc = G.map(&p.in[0].b0, 64)) return rc;
  if (const int rc = U.map(&p.in[0].b1, 64)) return rc;
  if (!dh) return run_product<T, kForward>(p, s);
  if (const int rc = run_product<T, kGates>(p, s)) return rc;
  const Operand D{p.gates, m, f, p.pitch, 2 * C::kPlanes};
  p.out = dx, p.dwg = dwg, p.dwu = dwu, p.parts = l.parts, p.splits = l.splits, p.split_steps = l.split_steps;
  p.dx_parts = l.dx_parts, p.dx_splits = l.dx_splits, p.dx_split_steps = l.dx_split_steps, p.extra = l.extra;
  p.col_tiles = tile_count(k, C::kCols);
  p.turned = turns(kDtype, k, f);
  p.weight_rows = tile_count(p.turned ? f : k, 2 * kRows), p.weight_cols = 2 * tile_count(p.turned ? k : f, C::kCols);
  if (const int rc = D.map(&p.in[0].a, kRows)) return rc;
  if (const int rc = G.map(&p.in[0].b0, C::kHalf)) return rc;
  if (const int rc = U.map(&p.in[0].b1, C::kHalf)) return rc;
  if (const int rc = (p.turned ? D : X).map(&p.in[1].a, 64)) return rc;
  if (const int rc = (p.turned ? X : D).map(&p.in[1].b0, 64)) return rc;
  if (const int rc = run_product<T, kGradients>(p, s)) return rc;
  const int64_t sums = (l.splits > 1 ? 2 * k * f : 0) + (l.dx_splits > 1 ? m * k : 0);
  if (sums == 0) return RLENV_OK;
  add_parts_kernel<T><<<grid_for(sums, 256), 256, 0, s>>>(l.parts, l.splits, k * f, static_cast<T*>(dwg), static_cast<T*>(dwu),
                                                         l.dx_parts, l.dx_splits, m * k, static_cast<T*>(dx));
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
  if (!out || !x || !w_gate || !w_up || off_boundary(x, w_gate, w_up) || off_boundary(out, out, out)) return RLENV_EINVAL;
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
  if (!grad_out || !x || !w_gate || !w_up || !grad_x || !grad_w_gate || !grad_w_up || off_boundary(x, w_gate, w_up) ||
      off_boundary(grad_x, grad_w_gate, grad_w_up))
    return RLENV_EINVAL;
  const Layout l = lay_out(dtype, m, k, f, true, scratch);
  if (!scratch_holds(scratch, scratch_bytes, l.bytes)) return RLENV_EINVAL;
  const cudaStream_t s = as_stream(stream);
  return dtype == RLENV_F32 ? ffn<float>(grad_out, x, w_gate, w_up, m, k, f, activation, nullptr, grad_x, grad_w_gate,
                                         grad_w_up, l, s)
                            : ffn<__nv_bfloat16>(grad_out, x, w_gate, w_up, m, k, f, activation, nullptr, grad_x,
                                                 grad_w_gate, grad_w_up, l, s);
}

int rlenv_gated_ffn_status(unsigned int* gave_up, int clear) {
  if (!gave_up) return RLENV_EINVAL;
  *gave_up = 0;
  return rlenv::bw::read_given_up(gave_up, clear != 0);
}

}  // extern "C"
