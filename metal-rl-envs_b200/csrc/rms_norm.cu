// Root-mean-square norm with the residual's addition, its gradient, and its output in 8-bit integers. For a row x of
// K values, a row y of the residual stream and weights w,
//     t = x + y,   r = (t't / K + eps)^(-1/2),   out = (t r) w,
// t rounded to the rows' type only where it is stored. With the gradients g of out and s of t,
//     dt = s + r (w g) - t r^3 ((w g)'t) / K,   dw = sum over rows of g (t r).
// In 8 bits a row is whole numbers, round(out 127 / max |out|), and the scale max |out| / 127.
//
// Bound by memory: each value is read once and written once, a row held in registers between its sums and its
// results. A row is a warp's or a block's: `Team`.
#include <cuda_bf16.h>

#include <type_traits>

#include "common.cuh"

namespace rlenv {
namespace {

// Values a thread moves at once: 16 bytes where every row starts on a 16-byte boundary and holds whole vectors, else
// one value (kWide false).
template <typename T, bool kWide>
struct Vec {
  static constexpr int kValues = kWide ? 16 / int(sizeof(T)) : 1;
};

// A vector as it lies in memory, and its values. Rows wait in registers in this form: half the room for bfloat16, and
// nothing that waits for a load while others are to be issued (bfloat16 rows of 333 by single values, the gradient of
// 100,000: 658 us when each was converted as it came).
template <typename T, bool kWide>
struct Raw {
  uint4 bits;
  RLENV_D void load(const T* from) { bits = __ldg(reinterpret_cast<const uint4*>(from)); }
  RLENV_D void clear() { bits = make_uint4(0, 0, 0, 0); }
  RLENV_D void values(float (&v)[16 / sizeof(T)]) const {
    const uint32_t w[4] = {bits.x, bits.y, bits.z, bits.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (sizeof(T) == 4)
        v[i] = __uint_as_float(w[i]);
      else
        v[2 * i] = __uint_as_float(w[i] << 16), v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
  }
};
template <>
struct Raw<float, false> {
  float bits;
  RLENV_D void load(const float* from) { bits = __ldg(from); }
  RLENV_D void clear() { bits = 0.0f; }
  RLENV_D void values(float (&v)[1]) const { v[0] = bits; }
};
template <>
struct Raw<__nv_bfloat16, false> {
  unsigned short bits;
  RLENV_D void load(const __nv_bfloat16* from) { bits = __ldg(reinterpret_cast<const unsigned short*>(from)); }
  RLENV_D void clear() { bits = 0; }
  RLENV_D void values(float (&v)[1]) const { v[0] = __uint_as_float(uint32_t(bits) << 16); }
};
template <typename T, int kValues>
RLENV_D void load(const T* from, float (&v)[kValues]) {
  Raw<T, (kValues > 1)> raw;
  raw.load(from);
  raw.values(v);
}
template <int kValues>
RLENV_D void store(float* to, const float (&v)[kValues]) {
  if constexpr (kValues == 1)
    to[0] = v[0];
  else
    *reinterpret_cast<float4*>(to) = make_float4(v[0], v[1], v[2], v[3]);
}
RLENV_D uint32_t pair_bits(float lo, float hi) {
  const __nv_bfloat162 p = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&p);
}
template <int kValues>
RLENV_D void store(__nv_bfloat16* to, const float (&v)[kValues]) {
  if constexpr (kValues == 1)
    to[0] = __float2bfloat16_rn(v[0]);
  else
    *reinterpret_cast<uint4*>(to) = make_uint4(pair_bits(v[0], v[1]), pair_bits(v[2], v[3]), pair_bits(v[4], v[5]),
                                               pair_bits(v[6], v[7]));
}
// Whole numbers of at most 127 in magnitude, as bytes.
RLENV_D uint32_t byte_of(float x) { return uint32_t(__float2int_rn(x)) & 0xffu; }
template <int kValues>
RLENV_D void store_codes(int8_t* to, const float (&v)[kValues]) {
  if constexpr (kValues == 1) {
    to[0] = int8_t(__float2int_rn(v[0]));
  } else {
    uint32_t w[kValues / 4];
#pragma unroll
    for (int i = 0; i < kValues / 4; ++i)
      w[i] = byte_of(v[4 * i]) | byte_of(v[4 * i + 1]) << 8 | byte_of(v[4 * i + 2]) << 16 | byte_of(v[4 * i + 3]) << 24;
    if constexpr (kValues == 4)
      *reinterpret_cast<uint32_t*>(to) = w[0];
    else
      *reinterpret_cast<uint2*>(to) = make_uint2(w[0], w[1]);
  }
}

// The threads that share a row: some of a warp, a warp, some warps of a block, or a block.
template <int kThreads>
struct Team {
  static constexpr int kBlock = kThreads < 256 ? 256 : kThreads;  // threads of a block
  static constexpr int kRows = kBlock / kThreads;                 // rows it works on at a time
  static constexpr int kWarps = kThreads < 32 ? 1 : kThreads / 32;
  static constexpr int kSpan = kThreads < 32 ? kThreads : 32;     // its lanes in a warp

  static RLENV_D void sync() {  // of more than a warp
    if constexpr (kRows == 1)
      __syncthreads();
    else
      asm volatile("bar.sync %0, %1;" ::"r"(int(threadIdx.x) / kThreads + 1), "n"(kThreads) : "memory");
  }
  // The sum over the team of each of kN values, in a fixed order; `room` holds kN kWarps of them for each team.
  template <int kN>
  static RLENV_D void sum(float (&v)[kN], float* room) {
#pragma unroll
    for (int i = 0; i < kN; ++i)
#pragma unroll
      for (int d = kSpan / 2; d > 0; d /= 2) v[i] += __shfl_xor_sync(0xffffffffu, v[i], d);
    if constexpr (kWarps > 1) {
      room += threadIdx.x / kThreads * (kN * kWarps);
      const int warp = threadIdx.x % kThreads / 32, lane = threadIdx.x % 32;
      sync();  // the room's last values are read
      if (lane == 0)
#pragma unroll
        for (int i = 0; i < kN; ++i) room[i * kWarps + warp] = v[i];
      sync();
#pragma unroll
      for (int i = 0; i < kN; ++i) {
        v[i] = room[i * kWarps + lane % kWarps];
#pragma unroll
        for (int d = kWarps / 2; d > 0; d /= 2) v[i] += __shfl_xor_sync(0xffffffffu, v[i], d);
      }
    }
  }
  // The largest of the team's whole numbers.
  static RLENV_D uint32_t largest(uint32_t v, uint32_t* room) {
#pragma unroll
    for (int d = kSpan / 2; d > 0; d /= 2) v = max(v, __shfl_xor_sync(0xffffffffu, v, d));
    if constexpr (kWarps > 1) {
      room += threadIdx.x / kThreads * kWarps;
      const int warp = threadIdx.x % kThreads / 32, lane = threadIdx.x % 32;
      sync();
      if (lane == 0) room[warp] = v;
      sync();
      v = __reduce_max_sync(0xffffffffu, room[lane % kWarps]);
    }
    return v;
  }
};

struct Norm {
  int64_t m, k;
  const void *x, *residual, *weight;  // residual and weight may be null
  int64_t x_stride, residual_stride;
  float eps;
  void *out, *total;  // total may be null
  int8_t* codes;      // 8-bit output: rows of `pitch` bytes, and their scales
  int64_t pitch;
  float* scale;
  bool normalise;     // 8-bit output: of the norm, or of x itself
};

// Rows whose largest magnitude is below this are zero in 8 bits: 127 / max is a float32 above it.
constexpr float kTiny = 0x1p-100f;

// Rows of at most kThreads kVectors vectors: kCodes false, out; true, codes and scale.
template <typename T, bool kWide, int kThreads, int kVectors, bool kCodes>
__global__ void __launch_bounds__(Team<kThreads>::kBlock) norm_kernel(const __grid_constant__ Norm p) {
  using G = Team<kThreads>;
  constexpr int kN = Vec<T, kWide>::kValues;
  __shared__ float room[G::kWarps * G::kRows];
  const int at = threadIdx.x % kThreads, k = int(p.k);
  const int64_t row = int64_t(blockIdx.x) * G::kRows + threadIdx.x / kThreads;
  const bool there = row < p.m;
  const T *x = static_cast<const T*>(p.x) + row * p.x_stride,
          *residual = p.residual ? static_cast<const T*>(p.residual) + row * p.residual_stride : nullptr,
          *weight = static_cast<const T*>(p.weight);
  const auto column = [&](int i) { return (at + i * kThreads) * kN; };
  const auto in = [&](int i) { return there && column(i) < k; };
  float t[kVectors][kN];
  Raw<T, kWide> from[kVectors], other[kVectors];
#pragma unroll
  for (int i = 0; i < kVectors; ++i) {
    from[i].clear();
    if (in(i)) from[i].load(x + column(i));
  }
  if (residual) {
#pragma unroll
    for (int i = 0; i < kVectors; ++i) {
      other[i].clear();
      if (in(i)) other[i].load(residual + column(i));
    }
  }
  float sum[1] = {0.0f};
#pragma unroll
  for (int i = 0; i < kVectors; ++i) {
    from[i].values(t[i]);
    if (residual) {
      float y[kN];
      other[i].values(y);
#pragma unroll
      for (int j = 0; j < kN; ++j) t[i][j] += y[j];
    }
#pragma unroll
    for (int j = 0; j < kN; ++j) sum[0] = fmaf(t[i][j], t[i][j], sum[0]);
  }
  if (weight) {  // on its way while the sum is formed
#pragma unroll
    for (int i = 0; i < kVectors; ++i)
      if (column(i) < k) other[i].load(weight + column(i));
  }
  if (p.total) {
    T* const total = static_cast<T*>(p.total) + row * p.k;
#pragma unroll
    for (int i = 0; i < kVectors; ++i)
      if (in(i)) store(total + column(i), t[i]);
  }
  float r = 1.0f;
  if (!kCodes || p.normalise) {
    G::sum(sum, room);
    r = rsqrtf(sum[0] / float(k) + p.eps);
  }
#pragma unroll
  for (int i = 0; i < kVectors; ++i) {
    float w[kN];
    if (weight && column(i) < k) other[i].values(w);
#pragma unroll
    for (int j = 0; j < kN; ++j) t[i][j] = weight && column(i) < k ? t[i][j] * r * w[j] : t[i][j] * r;
  }
  if constexpr (!kCodes) {
    T* const out = static_cast<T*>(p.out) + row * p.k;
#pragma unroll
    for (int i = 0; i < kVectors; ++i)
      if (in(i)) store(out + column(i), t[i]);
  } else {
    // As bits, magnitudes are ordered with infinity and NaN above all numbers.
    uint32_t most = 0;
#pragma unroll
    for (int i = 0; i < kVectors; ++i)
#pragma unroll
      for (int j = 0; j < kN; ++j) most = max(most, in(i) ? __float_as_uint(t[i][j]) & 0x7fffffffu : 0u);
    most = G::largest(most, reinterpret_cast<uint32_t*>(room));
    const float top = __uint_as_float(most);
    const bool some = top >= kTiny && most < 0x7f800000u;
    const float to_codes = some ? 127.0f / top : 0.0f;
    if (at == 0 && there) p.scale[row] = some ? top / 127.0f : top < kTiny ? 0.0f : __uint_as_float(0x7fffffffu);
    int8_t* const codes = p.codes + row * p.pitch;
#pragma unroll
    for (int i = 0; i < kVectors; ++i) {
#pragma unroll
      for (int j = 0; j < kN; ++j) t[i][j] = some ? t[i][j] * to_codes : 0.0f;
      if (in(i)) store_codes(codes + column(i), t[i]);
    }
  }
}

// Rows longer than registers hold: read again for each of a row's passes, from L2 as a rule.
constexpr int kLong = 1024;
template <typename T, bool kCodes>
__global__ void __launch_bounds__(kLong) long_norm_kernel(const __grid_constant__ Norm p) {
  using G = Team<kLong>;
  __shared__ float room[G::kWarps];
  const int64_t row = blockIdx.x;
  const T *x = static_cast<const T*>(p.x) + row * p.x_stride,
          *residual = p.residual ? static_cast<const T*>(p.residual) + row * p.residual_stride : nullptr,
          *weight = static_cast<const T*>(p.weight);
  const auto total_at = [&](int64_t c) {
    float t[1], y[1];
    load(x + c, t);
    if (residual) load(residual + c, y), t[0] += y[0];
    return t[0];
  };
  float r = 1.0f;
  if (!kCodes || p.normalise) {
    float sum[1] = {0.0f};
    for (int64_t c = threadIdx.x; c < p.k; c += kLong) {
      const float t = total_at(c);
      sum[0] = fmaf(t, t, sum[0]);
    }
    G::sum(sum, room);
    r = rsqrtf(sum[0] / float(p.k) + p.eps);
  }
  const auto out_at = [&](int64_t c) {
    float w[1];
    const float v = total_at(c) * r;
    if (!weight) return v;
    load(weight + c, w);
    return v * w[0];
  };
  if constexpr (kCodes) {
    uint32_t most = 0;
    for (int64_t c = threadIdx.x; c < p.k; c += kLong) most = max(most, __float_as_uint(out_at(c)) & 0x7fffffffu);
    most = G::largest(most, reinterpret_cast<uint32_t*>(room));
    const float top = __uint_as_float(most);
    const bool some = top >= kTiny && most < 0x7f800000u;
    const float to_codes = some ? 127.0f / top : 0.0f;
    if (threadIdx.x == 0) p.scale[row] = some ? top / 127.0f : top < kTiny ? 0.0f : __uint_as_float(0x7fffffffu);
    for (int64_t c = threadIdx.x; c < p.k; c += kLong) {
      const float v[1] = {some ? out_at(c) * to_codes : 0.0f};
      store_codes(p.codes + row * p.pitch + c, v);
    }
  }
  for (int64_t c = threadIdx.x; c < p.k; c += kLong) {
    if constexpr (!kCodes) {
      const float v[1] = {out_at(c)};
      store(static_cast<T*>(p.out) + row * p.k + c, v);
    }
    if (p.total) {
      const float v[1] = {total_at(c)};
      store(static_cast<T*>(p.total) + row * p.k + c, v);
    }
  }
}

struct NormGrad {
  int64_t m, k;
  const void *grad_out, *total, *weight, *grad_total;  // weight and grad_total may be null
  int64_t grad_out_stride, total_stride, grad_total_stride;
  float eps;
  void* grad;
  float* parts;  // (blocks, K): each block's sums over its rows of the weight's gradient; null: none asked for
};

// A team's next row is on its way while it works on one (kAhead: where registers allow).
template <typename T, bool kWide, int kThreads, int kVectors>
__global__ void __launch_bounds__(Team<kThreads>::kBlock) norm_grad_kernel(const __grid_constant__ NormGrad p) {
  using G = Team<kThreads>;
  using R = Raw<T, kWide>;
  constexpr int kN = Vec<T, kWide>::kValues;
  constexpr bool kAhead = kVectors * int(sizeof(R)) <= 32;
  __shared__ float room[2 * G::kWarps * G::kRows];
  const int at = threadIdx.x % kThreads, k = int(p.k);
  const auto column = [&](int i) { return (at + i * kThreads) * kN; };
  float dw[kVectors][kN];
  R w[kVectors];
#pragma unroll
  for (int i = 0; i < kVectors; ++i) {
    w[i].clear();
    if (p.weight && column(i) < k) w[i].load(static_cast<const T*>(p.weight) + column(i));
#pragma unroll
    for (int j = 0; j < kN; ++j) dw[i][j] = 0.0f;
  }
  const auto weighed = [&](int i, float (&g)[kN]) {
    if (!p.weight) return;
    float v[kN];
    w[i].values(v);
#pragma unroll
    for (int j = 0; j < kN; ++j) g[j] *= v[j];
  };
  R t[kVectors], g[kVectors], s[kVectors];
  const auto load_row = [&](int64_t row, R (&t)[kVectors], R (&g)[kVectors], R (&s)[kVectors]) {
    const T *total = static_cast<const T*>(p.total) + row * p.total_stride,
            *grad_out = static_cast<const T*>(p.grad_out) + row * p.grad_out_stride,
            *grad_total = static_cast<const T*>(p.grad_total) + row * p.grad_total_stride;
#pragma unroll
    for (int i = 0; i < kVectors; ++i) {
      t[i].clear(), g[i].clear(), s[i].clear();
      if (row < p.m && column(i) < k) {
        t[i].load(total + column(i));
        g[i].load(grad_out + column(i));
        if (p.grad_total) s[i].load(grad_total + column(i));
      }
    }
  };
  const int64_t step = int64_t(gridDim.x) * G::kRows;
  int64_t row = int64_t(blockIdx.x) * G::kRows + threadIdx.x / kThreads;
  // A warp's teams make as many turns as its first.
  const int64_t turns = (p.m - (int64_t(blockIdx.x) * G::kRows + threadIdx.x / 32 * 32 / kThreads) + step - 1) / step;
  if (kAhead) load_row(row, t, g, s);
  for (int64_t turn = 0; turn < turns; ++turn, row += step) {
    R next_t[kVectors], next_g[kVectors], next_s[kVectors];
    if (kAhead)
      load_row(row + step, next_t, next_g, next_s);
    else
      load_row(row, t, g, s);
    float sums[2] = {0.0f, 0.0f};
#pragma unroll
    for (int i = 0; i < kVectors; ++i) {
      float tv[kN], gv[kN];
      t[i].values(tv), g[i].values(gv);
      weighed(i, gv);
#pragma unroll
      for (int j = 0; j < kN; ++j) sums[0] = fmaf(tv[j], tv[j], sums[0]), sums[1] = fmaf(gv[j], tv[j], sums[1]);
    }
    G::sum(sums, room);
    const float r = rsqrtf(sums[0] / float(k) + p.eps), along = r * (r * sums[1] / float(k));
    T* const grad = static_cast<T*>(p.grad) + row * p.k;
#pragma unroll
    for (int i = 0; i < kVectors; ++i) {
      float tv[kN], gv[kN], v[kN];
      t[i].values(tv), g[i].values(gv), s[i].values(v);
#pragma unroll
      for (int j = 0; j < kN; ++j) dw[i][j] = fmaf(gv[j], tv[j] * r, dw[i][j]);
      weighed(i, gv);
#pragma unroll
      for (int j = 0; j < kN; ++j) v[j] += r * (gv[j] - tv[j] * along);
      if (row < p.m && column(i) < k) store(grad + column(i), v);
    }
    if (kAhead) {
#pragma unroll
      for (int i = 0; i < kVectors; ++i) t[i] = next_t[i], g[i] = next_g[i], s[i] = next_s[i];
    }
  }
  if (!p.parts) return;
  // A block's sums: the teams' of a warp, then the warps' one after the other, those of the same columns.
  if constexpr (kThreads < 32) {
#pragma unroll
    for (int i = 0; i < kVectors; ++i)
#pragma unroll
      for (int j = 0; j < kN; ++j)
#pragma unroll
        for (int d = kThreads; d < 32; d *= 2) dw[i][j] += __shfl_xor_sync(0xffffffffu, dw[i][j], d);
  }
  extern __shared__ float shared_dw[];
  constexpr int kSets = kThreads < 32 ? G::kBlock / 32 : G::kRows;  // of threads that share columns
  const int set = kThreads < 32 ? threadIdx.x / 32 : threadIdx.x / kThreads;
  for (int n = 0; n < kSets; ++n) {
    if (set == n && (kThreads >= 32 || threadIdx.x % 32 < kThreads)) {
#pragma unroll
      for (int i = 0; i < kVectors; ++i) {
#pragma unroll
        for (int j = 0; j < kN; ++j) {
          float* const to = shared_dw + (j * kVectors + i) * kThreads + at;
          if (n > 0) dw[i][j] += *to;
          if (n + 1 < kSets)
            *to = dw[i][j];
          else if (column(i) < k)
            p.parts[int64_t(blockIdx.x) * p.k + column(i) + j] = dw[i][j];
        }
      }
    }
    if (kSets > 1) __syncthreads();
  }
}

template <typename T>
__global__ void __launch_bounds__(kLong) long_norm_grad_kernel(const __grid_constant__ NormGrad p) {
  using G = Team<kLong>;
  __shared__ float room[2 * G::kWarps];
  const T* const weight = static_cast<const T*>(p.weight);
  float* const part = p.parts ? p.parts + int64_t(blockIdx.x) * p.k : nullptr;
  for (int64_t row = blockIdx.x; row < p.m; row += gridDim.x) {
    const T *total = static_cast<const T*>(p.total) + row * p.total_stride,
            *grad_out = static_cast<const T*>(p.grad_out) + row * p.grad_out_stride;
    float sums[2] = {0.0f, 0.0f}, t[1], g[1], w[1] = {1.0f};
    for (int64_t c = threadIdx.x; c < p.k; c += kLong) {
      load(total + c, t), load(grad_out + c, g);
      if (weight) load(weight + c, w);
      sums[0] = fmaf(t[0], t[0], sums[0]), sums[1] = fmaf(g[0] * w[0], t[0], sums[1]);
    }
    G::sum(sums, room);
    const float r = rsqrtf(sums[0] / float(p.k) + p.eps), along = r * (r * sums[1] / float(p.k));
    for (int64_t c = threadIdx.x; c < p.k; c += kLong) {
      load(total + c, t), load(grad_out + c, g);
      if (weight) load(weight + c, w);
      float v[1] = {r * (g[0] * w[0] - t[0] * along)}, s[1];
      if (p.grad_total) {
        load(static_cast<const T*>(p.grad_total) + row * p.grad_total_stride + c, s);
        v[0] += s[0];
      }
      store(static_cast<T*>(p.grad) + row * p.k + c, v);
      if (part) part[c] = fmaf(g[0], t[0] * r, row == blockIdx.x ? 0.0f : part[c]);
    }
  }
}

// The weight's gradient: the blocks' sums added up, a column by 32 threads in a fixed order.
template <typename T>
__global__ void __launch_bounds__(256) add_rows_kernel(const float* __restrict__ parts, int count, int64_t k,
                                                       T* __restrict__ grad_weight) {
  __shared__ float room[8][33];
  const int part = threadIdx.x / 8, column = threadIdx.x / 32;
  const int64_t c = int64_t(blockIdx.x) * 8 + threadIdx.x % 8, first = int64_t(blockIdx.x) * 8;
  float sum = 0.0f;
  if (c < k) {
#pragma unroll 8
    for (int i = part; i < count; i += 32) sum += __ldg(parts + i * k + c);
  }
  room[threadIdx.x % 8][part] = sum;
  __syncthreads();
  sum = room[column][threadIdx.x % 32];
#pragma unroll
  for (int d = 16; d > 0; d /= 2) sum += __shfl_xor_sync(0xffffffffu, sum, d);
  if (threadIdx.x % 32 == 0 && first + column < k) {
    const float v[1] = {sum};
    store(grad_weight + first + column, v);
  }
}

bool on16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

template <int kTeam, int kCount>
struct Form {
  static constexpr int kThreads = kTeam, kVectors = kCount;
};
// Calls f with the form for rows of `vectors` vectors; false where none holds them.
template <bool kWide, typename F>
bool with_form(int64_t vectors, F&& f) {
  if constexpr (kWide) {
    if (vectors <= 8) return f(Form<8, 1>()), true;
    if (vectors <= 16) return f(Form<16, 1>()), true;
    if (vectors <= 32) return f(Form<32, 1>()), true;
    if (vectors <= 64) return f(Form<32, 2>()), true;
    if (vectors <= 128) return f(Form<32, 4>()), true;
    if (vectors <= 512) return f(Form<128, 4>()), true;
    if (vectors <= 2048) return f(Form<512, 4>()), true;
    if (vectors <= 4096) return f(Form<512, 8>()), true;
  } else {
    if (vectors <= 32) return f(Form<32, 1>()), true;
    if (vectors <= 128) return f(Form<32, 4>()), true;
    if (vectors <= 256) return f(Form<32, 8>()), true;
    if (vectors <= 1024) return f(Form<128, 8>()), true;
    if (vectors <= 4096) return f(Form<512, 8>()), true;
    if (vectors <= 16384) return f(Form<1024, 16>()), true;
  }
  return false;
}
// The gradient holds three rows, the next three and the weight's gradient.
template <typename T, bool kWide, typename F>
bool with_grad_form(int64_t vectors, F&& f) {
  if constexpr (kWide) {
    if (vectors <= 8) return f(Form<8, 1>()), true;
    if (vectors <= 16) return f(Form<16, 1>()), true;
    if (vectors <= 32) return f(Form<32, 1>()), true;
    if (vectors <= 64) return f(Form<32, 2>()), true;
    if (vectors <= 128) return f(Form<64, 2>()), true;
    if (vectors <= 256) return f(Form<128, 2>()), true;
    if (vectors <= 512) return f(Form<256, 2>()), true;
    if (vectors <= 1024) return f(Form<512, 2>()), true;
    if (vectors <= 2048) return f(Form<512, 4>()), true;
    if (sizeof(T) == 4 && vectors <= 4096) return f(Form<512, 8>()), true;
  } else {
    if (vectors <= 32) return f(Form<32, 1>()), true;
    if (vectors <= 128) return f(Form<32, 4>()), true;
    if (vectors <= 256) return f(Form<32, 8>()), true;
    if (vectors <= 512) return f(Form<64, 8>()), true;
    if (vectors <= 1024) return f(Form<128, 8>()), true;
    if (vectors <= 2048) return f(Form<256, 8>()), true;
    if (vectors <= 4096) return f(Form<512, 8>()), true;
    if (vectors <= 8192) return f(Form<512, 16>()), true;
  }
  return false;
}

template <typename T, bool kCodes>
int norm(const Norm& p, cudaStream_t s) {
  constexpr int kN = 16 / int(sizeof(T));
  const bool wide = p.k % kN == 0 && on16(p.x) && on16(p.residual) && on16(p.weight) && on16(p.out) && on16(p.total) &&
                    p.x_stride % kN == 0 && p.residual_stride % kN == 0 && (!kCodes || (on16(p.codes) && p.pitch % 16 == 0));
  bool held;
  if (wide)
    held = with_form<true>(p.k / kN, [&](auto form) {
      using G = Team<form.kThreads>;
      norm_kernel<T, true, form.kThreads, form.kVectors, kCodes><<<unsigned((p.m + G::kRows - 1) / G::kRows), G::kBlock, 0, s>>>(p);
    });
  else
    held = with_form<false>(p.k, [&](auto form) {
      using G = Team<form.kThreads>;
      norm_kernel<T, false, form.kThreads, form.kVectors, kCodes><<<unsigned((p.m + G::kRows - 1) / G::kRows), G::kBlock, 0, s>>>(p);
    });
  if (!held) long_norm_kernel<T, kCodes><<<unsigned(p.m), kLong, 0, s>>>(p);
  return launch_status();
}

constexpr int kGradBlocks = 2 * 148;
// Blocks of the gradient's kernel, each with a row of the weight's gradient in scratch.
int64_t grad_blocks(int64_t m) { return m < kGradBlocks ? m : kGradBlocks; }

template <typename T>
int norm_grad(const NormGrad& p, void* grad_weight, cudaStream_t s) {
  constexpr int kN = 16 / int(sizeof(T));
  const bool wide = p.k % kN == 0 && on16(p.grad_out) && on16(p.total) && on16(p.weight) && on16(p.grad_total) &&
                    on16(p.grad) && p.grad_out_stride % kN == 0 && p.total_stride % kN == 0 && p.grad_total_stride % kN == 0;
  int64_t blocks = grad_blocks(p.m);
  bool held;
  const auto launch = [&](auto form, auto is_wide) {
    constexpr bool kWide = decltype(is_wide)::value;
    using G = Team<form.kThreads>;
    blocks = grad_blocks((p.m + G::kRows - 1) / G::kRows);
    const size_t shared = G::kRows > 1 ? form.kThreads * form.kVectors * Vec<T, kWide>::kValues * sizeof(float) : 0;  // the warps' sums
    norm_grad_kernel<T, kWide, form.kThreads, form.kVectors><<<unsigned(blocks), G::kBlock, shared, s>>>(p);
  };
  if (wide)
    held = with_grad_form<T, true>(p.k / kN, [&](auto form) { launch(form, std::true_type()); });
  else
    held = with_grad_form<T, false>(p.k, [&](auto form) { launch(form, std::false_type()); });
  if (!held) long_norm_grad_kernel<T><<<unsigned(blocks), kLong, 0, s>>>(p);
  if (int rc = launch_status(); rc || !p.parts) return rc;
  add_rows_kernel<T><<<unsigned((p.k + 7) / 8), 256, 0, s>>>(p.parts, int(blocks), p.k, static_cast<T*>(grad_weight));
  return launch_status();
}

bool norm_sizes(int dtype, int64_t m, int64_t k) {
  return (dtype == RLENV_F32 || dtype == RLENV_BF16) && m >= 0 && k >= 1 && m < (int64_t(1) << 31) && k < (int64_t(1) << 31);
}
// Rows of `size`-byte values at p, `stride` apart (0: one row for all).
bool rows_fit(const void* p, int64_t stride, int size) {
  return stride >= 0 && reinterpret_cast<uintptr_t>(p) % size == 0;
}

}  // namespace
}  // namespace rlenv

extern "C" {

int rlenv_rms_norm_forward(int dtype, int64_t m, int64_t k, const void* x, int64_t x_stride, const void* residual,
                           int64_t residual_stride, const void* weight, float eps, void* out, void* total, void* stream) {
  using namespace rlenv;
  if (!norm_sizes(dtype, m, k) || !(eps >= 0.0f)) return RLENV_EINVAL;
  if (m == 0) return RLENV_OK;
  const int size = dtype == RLENV_F32 ? 4 : 2;
  if (!x || !out || !rows_fit(x, x_stride, size) || !rows_fit(residual, residual_stride, size) ||
      !rows_fit(weight, 0, size) || !rows_fit(out, 0, size) || !rows_fit(total, 0, size))
    return RLENV_EINVAL;
  const Norm p{m, k, x, residual, weight, x_stride, residual ? residual_stride : 0, eps, out, total, nullptr, 0, nullptr, true};
  return dtype == RLENV_F32 ? norm<float, false>(p, as_stream(stream)) : norm<__nv_bfloat16, false>(p, as_stream(stream));
}

int rlenv_rms_norm_codes(int dtype, int64_t m, int64_t k, const void* x, int64_t x_stride, const void* residual,
                         int64_t residual_stride, const void* weight, float eps, int normalise, int8_t* codes,
                         int64_t pitch, float* scale, void* total, void* stream) {
  using namespace rlenv;
  if (!norm_sizes(dtype, m, k) || !(eps >= 0.0f) || pitch < k) return RLENV_EINVAL;
  if (m == 0) return RLENV_OK;
  const int size = dtype == RLENV_F32 ? 4 : 2;
  if (!x || !codes || !scale || !rows_fit(x, x_stride, size) || !rows_fit(residual, residual_stride, size) ||
      !rows_fit(weight, 0, size) || !rows_fit(scale, 0, 4) || !rows_fit(total, 0, size))
    return RLENV_EINVAL;
  const Norm p{m, k, x, residual, weight, x_stride, residual ? residual_stride : 0, eps, nullptr, total, codes, pitch, scale,
               normalise != 0};
  return dtype == RLENV_F32 ? norm<float, true>(p, as_stream(stream)) : norm<__nv_bfloat16, true>(p, as_stream(stream));
}

int64_t rlenv_rms_norm_scratch_bytes(int64_t m, int64_t k) {
  using namespace rlenv;
  if (!norm_sizes(RLENV_F32, m, k)) return RLENV_EINVAL;
  return grad_blocks(m) * k * 4;
}

int rlenv_rms_norm_backward(int dtype, int64_t m, int64_t k, const void* grad_out, int64_t grad_out_stride, const void* total,
                            int64_t total_stride, const void* weight, float eps, const void* grad_total,
                            int64_t grad_total_stride, void* grad, void* grad_weight, void* scratch, int64_t scratch_bytes,
                            void* stream) {
  using namespace rlenv;
  if (!norm_sizes(dtype, m, k) || !(eps >= 0.0f)) return RLENV_EINVAL;
  if (m == 0) return grad_weight ? RLENV_EINVAL : RLENV_OK;  // a sum over no rows is the caller's to fill
  const int size = dtype == RLENV_F32 ? 4 : 2;
  if (!grad_out || !total || !grad || !rows_fit(grad_out, grad_out_stride, size) || !rows_fit(total, total_stride, size) ||
      !rows_fit(weight, 0, size) || !rows_fit(grad_total, grad_total_stride, size) || !rows_fit(grad, 0, size) ||
      !rows_fit(grad_weight, 0, size))
    return RLENV_EINVAL;
  if (grad_weight && !scratch_holds(scratch, scratch_bytes, rlenv_rms_norm_scratch_bytes(m, k))) return RLENV_EINVAL;
  const NormGrad p{m, k, grad_out, total, weight, grad_total, grad_out_stride, total_stride, grad_total ? grad_total_stride : 0,
                   eps, grad, grad_weight ? static_cast<float*>(scratch) : nullptr};
  return dtype == RLENV_F32 ? norm_grad<float>(p, grad_weight, as_stream(stream))
                            : norm_grad<__nv_bfloat16>(p, grad_weight, as_stream(stream));
}

}  // extern "C"
