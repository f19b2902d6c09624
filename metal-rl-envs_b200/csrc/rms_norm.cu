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

#include <initializer_list>
#include <type_traits>

#include "common.cuh"

namespace rlenv {
namespace {

// How a row is moved. kWhole: vectors of 16 bytes, where every row starts on a 16-byte boundary and holds whole ones.
// kSkewed: rows of any length whose tensors all lie alike on the boundaries: vectors between the first boundary in the row
// and the last, and the up to 14 values before and after them by a lane each (bfloat16 rows of 333, 100,000 forward 60 us,
// by single values 182). kSingle: one value at a time.
enum Way { kWhole, kSkewed, kSingle };
template <typename T, Way kWay>
struct Vec {
  static constexpr int kValues = kWay == kSingle ? 1 : 16 / int(sizeof(T));
};

// A vector as it lies in memory, and its values. Rows wait in registers in this form: half the room for bfloat16, and
// nothing that waits for a load while others are to be issued.
template <typename T, int kValues>
struct Raw {
  uint4 bits;
  RLENV_D void load(const T* from) { bits = __ldg(reinterpret_cast<const uint4*>(from)); }
  RLENV_D void clear() { bits = make_uint4(0, 0, 0, 0); }
  RLENV_D void values(float* v) const {
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
struct Raw<float, 1> {
  float bits;
  RLENV_D void load(const float* from) { bits = __ldg(from); }
  RLENV_D void clear() { bits = 0.0f; }
  RLENV_D void values(float* v) const { v[0] = bits; }
};
template <>
struct Raw<__nv_bfloat16, 1> {
  unsigned short bits;
  RLENV_D void load(const __nv_bfloat16* from) { bits = __ldg(reinterpret_cast<const unsigned short*>(from)); }
  RLENV_D void clear() { bits = 0; }
  RLENV_D void values(float* v) const { v[0] = __uint_as_float(uint32_t(bits) << 16); }
};
// A vector from any place, as the words that hold it: those of bfloat16 start a value earlier where that lies on a boundary of
// four bytes. `from` itself may be the array's first value only where it lies on one.
template <typename T>
struct Between {
  static constexpr int kWords = sizeof(T) == 2 ? 5 : 4;
  uint32_t words[kWords];
  RLENV_D void clear() {
#pragma unroll
    for (int i = 0; i < kWords; ++i) words[i] = 0;
  }
  RLENV_D void load(const T* from, bool between) {
    const uint32_t* const at = reinterpret_cast<const uint32_t*>(between ? from - 1 : from);
#pragma unroll
    for (int i = 0; i < 4; ++i) words[i] = __ldg(at + i);
    if constexpr (kWords == 5) words[4] = __ldg(reinterpret_cast<const unsigned short*>(from) + 7);
  }
  RLENV_D uint4 bits(bool between) const {
    if constexpr (kWords == 4) return make_uint4(words[0], words[1], words[2], words[3]);
    const int by = between ? 16 : 0;
    return make_uint4(__funnelshift_r(words[0], words[1], by), __funnelshift_r(words[1], words[2], by),
                      __funnelshift_r(words[2], words[3], by), __funnelshift_r(words[3], words[kWords - 1], by));
  }
};
template <typename T>
RLENV_D float load(const T* from) {
  Raw<T, 1> raw;
  float v;
  raw.load(from);
  raw.values(&v);
  return v;
}
RLENV_D uint32_t pair_bits(float lo, float hi) {
  const __nv_bfloat162 p = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&p);
}
RLENV_D void store(float* to, float v) { *to = v; }
RLENV_D void store(__nv_bfloat16* to, float v) { *to = __float2bfloat16_rn(v); }
RLENV_D void store(int8_t* to, float v) { *to = int8_t(__float2int_rn(v)); }  // a whole number of at most 127
RLENV_D void store_vector(float* to, const float* v) { *reinterpret_cast<float4*>(to) = make_float4(v[0], v[1], v[2], v[3]); }
RLENV_D void store_vector(__nv_bfloat16* to, const float* v) {
  *reinterpret_cast<uint4*>(to) =
      make_uint4(pair_bits(v[0], v[1]), pair_bits(v[2], v[3]), pair_bits(v[4], v[5]), pair_bits(v[6], v[7]));
}
RLENV_D uint32_t byte_of(float x) { return uint32_t(__float2int_rn(x)) & 0xffu; }
template <int kValues>
RLENV_D void store_bytes(int8_t* to, const float* v) {  // on a boundary of kValues bytes
  uint32_t w[kValues / 4];
#pragma unroll
  for (int i = 0; i < kValues / 4; ++i)
    w[i] = byte_of(v[4 * i]) | byte_of(v[4 * i + 1]) << 8 | byte_of(v[4 * i + 2]) << 16 | byte_of(v[4 * i + 3]) << 24;
  if constexpr (kValues == 4)
    *reinterpret_cast<uint32_t*>(to) = w[0];
  else
    *reinterpret_cast<uint2*>(to) = make_uint2(w[0], w[1]);
}

// A thread's part of a row of k values: kVectors vectors, kThreads vectors apart, and with kSkewed one value more. All its
// values lie side by side in arrays of kCount.
template <typename T, Way kWay, int kThreads, int kVectors>
struct Part {
  static constexpr int kN = Vec<T, kWay>::kValues, kEdge = kWay == kSkewed, kCount = kVectors * kN + kEdge;
  struct Row {
    Raw<T, kN> vectors[kVectors];
    Raw<T, 1> edge;
    RLENV_D void values(float (&v)[kCount]) const {
#pragma unroll
      for (int i = 0; i < kVectors; ++i) vectors[i].values(v + i * kN);
      if constexpr (kEdge) edge.values(v + kVectors * kN);
    }
  };
  int k, first, count, edge;  // the first vector's place, how many this thread has, the single value's place or -1
  // of a row at `row`, as far as that lies on the boundaries
  RLENV_D Part(const void* row, int k, int at) : k(k), edge(-1) {
    int head = 0;
    if constexpr (kEdge) head = min(k, (16 - int(reinterpret_cast<uintptr_t>(row) % 16)) % 16 / int(sizeof(T)));
    const int vectors = (k - head) / kN, tail = k - head - vectors * kN;
    first = head + at * kN;
    count = at < vectors ? (vectors - at + kThreads - 1) / kThreads : 0;
    if constexpr (kEdge) edge = at < head ? at : at >= kN && at - kN < tail ? head + vectors * kN + at - kN : -1;
  }
  RLENV_D int place(int i) const { return first + i * kThreads * kN; }
  RLENV_D void load(const T* row, Row& r) const {
#pragma unroll
    for (int i = 0; i < kVectors; ++i) {
      r.vectors[i].clear();
      if (i < count) r.vectors[i].load(row + place(i));
    }
    if constexpr (kEdge) {
      r.edge.clear();
      if (edge >= 0) r.edge.load(row + edge);
    }
  }
  RLENV_D void fetch(const T* row) const {  // into L2
#pragma unroll
    for (int i = 0; i < kVectors; ++i)
      if (i < count) asm volatile("prefetch.global.L2 [%0];" ::"l"(row + place(i)));
  }
  RLENV_D void clear(Row& r) const {
#pragma unroll
    for (int i = 0; i < kVectors; ++i) r.vectors[i].clear();
    r.edge.clear();
  }
  // The weights of these places: they lie on a boundary by themselves, so that a skewed row's vectors of them do not. Nothing
  // waits for them before `values`.
  struct Weights {
    std::conditional_t<kEdge, Between<T>, Raw<T, kN>> vectors[kVectors];
    Raw<T, 1> edge;
    bool between;
    RLENV_D Row row() const {
      Row r;
#pragma unroll
      for (int i = 0; i < kVectors; ++i) {
        if constexpr (kEdge)
          r.vectors[i].bits = vectors[i].bits(between);
        else
          r.vectors[i] = vectors[i];
      }
      if constexpr (kEdge) r.edge = edge;
      return r;
    }
  };
  RLENV_D void load_weight(const T* weight, Weights& r) const {
    r.between = kEdge && sizeof(T) == 2 && first % 2;
#pragma unroll
    for (int i = 0; i < kVectors; ++i) {
      r.vectors[i].clear();
      if (i < count) {
        if constexpr (kEdge)
          r.vectors[i].load(weight + place(i), r.between);
        else
          r.vectors[i].load(weight + place(i));
      }
    }
    if constexpr (kEdge) {
      r.edge.clear();
      if (edge >= 0) r.edge.load(weight + edge);
    }
  }
  RLENV_D void store_row(T* row, const float (&v)[kCount]) const {
#pragma unroll
    for (int i = 0; i < kVectors; ++i)
      if (i < count) {
        if constexpr (kN == 1)
          store(row + place(i), v[i]);
        else
          store_vector(row + place(i), v + i * kN);
      }
    if constexpr (kEdge)
      if (edge >= 0) store(row + edge, v[kVectors * kN]);
  }
  RLENV_D void store_codes(int8_t* row, const float (&v)[kCount]) const {
#pragma unroll
    for (int i = 0; i < kVectors; ++i)
      if (i < count) {
        if constexpr (kWay == kWhole) {
          store_bytes<kN>(row + place(i), v + i * kN);
        } else {  // off the codes' boundaries: 99,900 x 1,001 bf16 123 us, 16 bits out 85
#pragma unroll
          for (int j = 0; j < kN; ++j) store(row + place(i) + j, v[i * kN + j]);
        }
      }
    if constexpr (kEdge)
      if (edge >= 0) store(row + edge, v[kVectors * kN]);
  }
  // f(place, value) for what is there.
  template <typename F>
  RLENV_D void each(float (&v)[kCount], F&& f) const {
#pragma unroll
    for (int i = 0; i < kVectors; ++i)
      if (i < count) {
#pragma unroll
        for (int j = 0; j < kN; ++j) f(place(i) + j, v[i * kN + j]);
      }
    if constexpr (kEdge)
      if (edge >= 0) f(edge, v[kVectors * kN]);
  }
};

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
template <typename T, Way kWay, int kThreads, int kVectors, bool kCodes>
__global__ void __launch_bounds__(Team<kThreads>::kBlock) norm_kernel(const __grid_constant__ Norm p) {
  using G = Team<kThreads>;
  using P = Part<T, kWay, kThreads, kVectors>;
  constexpr int kCount = P::kCount;
  __shared__ float room[G::kWarps * G::kRows];
  const int at = threadIdx.x % kThreads;
  const int64_t row = int64_t(blockIdx.x) * G::kRows + threadIdx.x / kThreads;
  const bool there = row < p.m;
  const T *x = static_cast<const T*>(p.x) + row * p.x_stride,
          *residual = p.residual ? static_cast<const T*>(p.residual) + row * p.residual_stride : nullptr,
          *weight = static_cast<const T*>(p.weight);
  const P part(x, there ? int(p.k) : 0, at);
  typename P::Row from, other;
  part.load(x, from);
  if (residual) part.load(residual, other);
  float t[kCount], sum[1] = {0.0f};
  from.values(t);
  if (residual) {
    float y[kCount];
    other.values(y);
#pragma unroll
    for (int i = 0; i < kCount; ++i) t[i] += y[i];
  }
#pragma unroll
  for (int i = 0; i < kCount; ++i) sum[0] = fmaf(t[i], t[i], sum[0]);
  typename P::Weights weights;
  if (weight) part.load_weight(weight, weights);  // on its way while the sum is formed
  if (p.total && there) part.store_row(static_cast<T*>(p.total) + row * p.k, t);
  float r = 1.0f;
  if (!kCodes || p.normalise) {
    G::sum(sum, room);
    r = rsqrtf(sum[0] / float(p.k) + p.eps);
  }
#pragma unroll
  for (int i = 0; i < kCount; ++i) t[i] *= r;
  if (weight) {
    float w[kCount];
    weights.row().values(w);
#pragma unroll
    for (int i = 0; i < kCount; ++i) t[i] *= w[i];
  }
  if constexpr (!kCodes) {
    if (there) part.store_row(static_cast<T*>(p.out) + row * p.k, t);
  } else {
    // As bits, magnitudes are ordered with infinity and NaN above all numbers.
    uint32_t most = 0;
    part.each(t, [&](int, float v) { most = max(most, __float_as_uint(v) & 0x7fffffffu); });
    most = G::largest(most, reinterpret_cast<uint32_t*>(room));
    const float top = __uint_as_float(most);
    const bool some = top >= kTiny && most < 0x7f800000u;
    const float to_codes = some ? 127.0f / top : 0.0f;
    if (at == 0 && there) p.scale[row] = some ? top / 127.0f : top < kTiny ? 0.0f : __uint_as_float(0x7fffffffu);
#pragma unroll
    for (int i = 0; i < kCount; ++i) t[i] = some ? t[i] * to_codes : 0.0f;
    if (there) part.store_codes(p.codes + row * p.pitch, t);
  }
}

// Rows longer than registers hold: read again for each of a row's passes, from L2 as a rule, by single values: 400 MB in all
// of rows of 20,000 float32 105 us, 40,000 bf16 179 (at a copy's rate 61). 8-bit output looks at a row three times: of 40,000
// bf16 263 us.
constexpr int kLong = 1024;
template <typename T, bool kCodes>
__global__ void __launch_bounds__(kLong) long_norm_kernel(const __grid_constant__ Norm p) {
  using G = Team<kLong>;
  __shared__ float room[G::kWarps];
  const int64_t row = blockIdx.x;
  const T *x = static_cast<const T*>(p.x) + row * p.x_stride,
          *residual = p.residual ? static_cast<const T*>(p.residual) + row * p.residual_stride : nullptr,
          *weight = static_cast<const T*>(p.weight);
  const auto total_at = [&](int64_t c) { return residual ? load(x + c) + load(residual + c) : load(x + c); };
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
  const auto out_at = [&](int64_t c) { return weight ? total_at(c) * r * load(weight + c) : total_at(c) * r; };
  if constexpr (kCodes) {
    uint32_t most = 0;
    for (int64_t c = threadIdx.x; c < p.k; c += kLong) most = max(most, __float_as_uint(out_at(c)) & 0x7fffffffu);
    most = G::largest(most, reinterpret_cast<uint32_t*>(room));
    const float top = __uint_as_float(most);
    const bool some = top >= kTiny && most < 0x7f800000u;
    const float to_codes = some ? 127.0f / top : 0.0f;
    if (threadIdx.x == 0) p.scale[row] = some ? top / 127.0f : top < kTiny ? 0.0f : __uint_as_float(0x7fffffffu);
    for (int64_t c = threadIdx.x; c < p.k; c += kLong) store(p.codes + row * p.pitch + c, some ? out_at(c) * to_codes : 0.0f);
  }
  for (int64_t c = threadIdx.x; c < p.k; c += kLong) {
    if constexpr (!kCodes) store(static_cast<T*>(p.out) + row * p.k + c, out_at(c));
    if (p.total) store(static_cast<T*>(p.total) + row * p.k + c, total_at(c));
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

// A team's next row is on its way while it works on one (kAhead: where registers allow; else it is fetched into L2). Its rows are
// a multiple of 8 apart, so that they all lie alike on the boundaries. The longest rows' weight gradient lies in shared memory
// (kApart), a thread's columns in places of its own, and float32 weights are read from L1 for each use: 400 MB of rows of 16,384
// bf16 102 us, of 12,288 float32 91 (with all of it in registers, which do not hold it, 136 and 133; the next row on its way into
// shared memory too gains 5% there and costs 6,145 float32 20%). Two blocks of 256 threads an SM are what the grid
// counts on, also where a few values are spilled for it (rows of 641 bf16 104 us, else 124).
template <typename T, Way kWay, int kThreads, int kVectors>
struct Grads {
  using P = Part<T, kWay, kThreads, kVectors>;
  static constexpr bool kAhead = kVectors * int(sizeof(Raw<T, P::kN>)) <= 32, kApart = kWay != kSingle && kVectors * P::kN >= 32,
                        kHeldWeights = kVectors * int(sizeof(Raw<T, P::kN>)) <= 64;
  static constexpr int kApartBytes = kApart ? kThreads * kVectors * P::kN * 4 : 0;
  static constexpr int kBlocks = Team<kThreads>::kBlock <= 256 ? 2 : 1;  // an SM's, which the grid counts on
};
template <typename T, Way kWay, int kThreads, int kVectors>
__global__ void __launch_bounds__(Team<kThreads>::kBlock, (Grads<T, kWay, kThreads, kVectors>::kBlocks))
norm_grad_kernel(const __grid_constant__ NormGrad p) {
  using G = Team<kThreads>;
  using P = Part<T, kWay, kThreads, kVectors>;
  using Row = typename P::Row;
  using Form = Grads<T, kWay, kThreads, kVectors>;
  constexpr int kCount = P::kCount, kN = P::kN;
  constexpr bool kAhead = Form::kAhead, kApart = Form::kApart;
  constexpr int kOwn = kApart ? P::kEdge + 1 : kCount;  // columns whose sums are in registers
  extern __shared__ __align__(16) float columns[];
  __shared__ float room[2 * G::kWarps * G::kRows];
  const int at = threadIdx.x % kThreads, k = int(p.k);
  const int64_t step = int64_t(gridDim.x) * G::kRows;
  int64_t row = int64_t(blockIdx.x) * G::kRows + threadIdx.x / kThreads;
  // A warp's teams make as many turns as its first.
  const int64_t turns = (p.m - (int64_t(blockIdx.x) * G::kRows + threadIdx.x / 32 * 32 / kThreads) + step - 1) / step;
  const P part(static_cast<const T*>(p.total) + row * p.total_stride, k, at);
  float dw[kOwn];
#pragma unroll
  for (int i = 0; i < kOwn; ++i) dw[i] = 0.0f;
  const auto apart = [&](int i, int j) { return reinterpret_cast<float4*>(columns) + (i * (kN / 4) + j) * kThreads + at; };
  if constexpr (kApart) {
#pragma unroll
    for (int i = 0; i < kVectors; ++i)
#pragma unroll
      for (int j = 0; j < kN / 4; ++j) *apart(i, j) = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  }
  Row w, t, g, s;
  const auto load_weights = [&] {
    typename P::Weights weights;
    part.load_weight(static_cast<const T*>(p.weight), weights);
    w = weights.row();
  };
  if (p.weight && Form::kHeldWeights) load_weights();
  const auto weighed = [&](float (&v)[kCount]) {
    if (!p.weight) return;
    if (!Form::kHeldWeights) load_weights();
    float of[kCount];
    w.values(of);
#pragma unroll
    for (int i = 0; i < kCount; ++i) v[i] *= of[i];
  };
  const auto load_row = [&](int64_t row, Row& t, Row& g, Row& s) {
    if (row < p.m) {
      part.load(static_cast<const T*>(p.total) + row * p.total_stride, t);
      part.load(static_cast<const T*>(p.grad_out) + row * p.grad_out_stride, g);
      if (p.grad_total)
        part.load(static_cast<const T*>(p.grad_total) + row * p.grad_total_stride, s);
      else
        part.clear(s);
    } else {
      part.clear(t), part.clear(g), part.clear(s);
    }
  };
  if (kAhead) load_row(row, t, g, s);
  for (int64_t turn = 0; turn < turns; ++turn, row += step) {
    Row next_t, next_g, next_s;
    if (kAhead) {
      load_row(row + step, next_t, next_g, next_s);
    } else {
      load_row(row, t, g, s);
      if (kWay != kSingle && row + step < p.m) {
        part.fetch(static_cast<const T*>(p.total) + (row + step) * p.total_stride);
        part.fetch(static_cast<const T*>(p.grad_out) + (row + step) * p.grad_out_stride);
        if (p.grad_total) part.fetch(static_cast<const T*>(p.grad_total) + (row + step) * p.grad_total_stride);
      }
    }
    float tv[kCount], gv[kCount], sums[2] = {0.0f, 0.0f};
    t.values(tv), g.values(gv);
    weighed(gv);
#pragma unroll
    for (int i = 0; i < kCount; ++i) sums[0] = fmaf(tv[i], tv[i], sums[0]), sums[1] = fmaf(gv[i], tv[i], sums[1]);
    G::sum(sums, room);
    const float r = row < p.m ? rsqrtf(sums[0] / float(k) + p.eps) : 0.0f, along = r * (r * sums[1] / float(k));
    float v[kCount];
    t.values(tv), g.values(gv), s.values(v);
    if constexpr (kApart) {
#pragma unroll
      for (int i = 0; i < kVectors; ++i)
#pragma unroll
        for (int j = 0; j < kN / 4; ++j) {
          float4 sum = *apart(i, j);
          const int c = i * kN + 4 * j;
          sum.x = fmaf(gv[c], tv[c] * r, sum.x), sum.y = fmaf(gv[c + 1], tv[c + 1] * r, sum.y);
          sum.z = fmaf(gv[c + 2], tv[c + 2] * r, sum.z), sum.w = fmaf(gv[c + 3], tv[c + 3] * r, sum.w);
          *apart(i, j) = sum;
        }
      if constexpr (P::kEdge) dw[0] = fmaf(gv[kCount - 1], tv[kCount - 1] * r, dw[0]);
    } else {
#pragma unroll
      for (int i = 0; i < kCount; ++i) dw[i] = fmaf(gv[i], tv[i] * r, dw[i]);
    }
    weighed(gv);
#pragma unroll
    for (int i = 0; i < kCount; ++i) v[i] += r * (gv[i] - tv[i] * along);
    if (row < p.m) part.store_row(static_cast<T*>(p.grad) + row * p.k, v);
    if (kAhead) t = next_t, g = next_g, s = next_s;
  }
  if (!p.parts) return;
  // A block's sums: the teams' of a warp, then the warps' one after the other.
  if constexpr (kThreads < 32) {
#pragma unroll
    for (int i = 0; i < kCount; ++i)
#pragma unroll
      for (int d = kThreads; d < 32; d *= 2) dw[i] += __shfl_xor_sync(0xffffffffu, dw[i], d);
  }
  float* const block_part = p.parts + int64_t(blockIdx.x) * p.k;
  if constexpr (kApart) {
    static_assert(G::kRows == 1, "a block has one set of columns");
#pragma unroll
    for (int i = 0; i < kVectors; ++i)
      if (i < part.count) {
#pragma unroll
        for (int j = 0; j < kN / 4; ++j) {
          const float4 sum = *apart(i, j);
          float* const to = block_part + part.place(i) + 4 * j;
          to[0] = sum.x, to[1] = sum.y, to[2] = sum.z, to[3] = sum.w;
        }
      }
    if constexpr (P::kEdge)
      if (part.edge >= 0) block_part[part.edge] = dw[0];
  } else {
    constexpr int kSets = kThreads < 32 ? G::kBlock / 32 : G::kRows;  // of threads with all of the columns
    const int set = kThreads < 32 ? threadIdx.x / 32 : threadIdx.x / kThreads;
    for (int n = 0; n < kSets; ++n) {
      if (set == n && (kThreads >= 32 || threadIdx.x % 32 < kThreads)) {
        if (n > 0) part.each(dw, [&](int c, float& v) { v += columns[c]; });
        float* const to = n + 1 < kSets ? columns : block_part;
        if constexpr (kWay == kWhole) {
#pragma unroll
          for (int i = 0; i < kVectors; ++i)
            if (i < part.count) {
#pragma unroll
              for (int j = 0; j < kN; j += 4) store_vector(to + part.place(i) + j, dw + i * kN + j);
            }
        } else {
          part.each(dw, [&](int c, float v) { to[c] = v; });
        }
      }
      if (kSets > 1) __syncthreads();
    }
  }
}

// Three tensors' 400 MB of rows of 20,000 float32 162 us, 16,392 bf16 218, 32,768 bf16 303 (at a copy's rate 61).
template <typename T>
__global__ void __launch_bounds__(kLong) long_norm_grad_kernel(const __grid_constant__ NormGrad p) {
  using G = Team<kLong>;
  __shared__ float room[2 * G::kWarps];
  const T* const weight = static_cast<const T*>(p.weight);
  float* const part = p.parts ? p.parts + int64_t(blockIdx.x) * p.k : nullptr;
  for (int64_t row = blockIdx.x; row < p.m; row += gridDim.x) {
    const T *total = static_cast<const T*>(p.total) + row * p.total_stride,
            *grad_out = static_cast<const T*>(p.grad_out) + row * p.grad_out_stride,
            *grad_total = p.grad_total ? static_cast<const T*>(p.grad_total) + row * p.grad_total_stride : nullptr;
    const auto weighed_at = [&](int64_t c) { return weight ? load(grad_out + c) * load(weight + c) : load(grad_out + c); };
    float sums[2] = {0.0f, 0.0f};
    for (int64_t c = threadIdx.x; c < p.k; c += kLong) {
      const float t = load(total + c);
      sums[0] = fmaf(t, t, sums[0]), sums[1] = fmaf(weighed_at(c), t, sums[1]);
    }
    G::sum(sums, room);
    const float r = rsqrtf(sums[0] / float(p.k) + p.eps), along = r * (r * sums[1] / float(p.k));
    for (int64_t c = threadIdx.x; c < p.k; c += kLong) {
      const float t = load(total + c), v = r * (weighed_at(c) - t * along);
      store(static_cast<T*>(p.grad) + row * p.k + c, grad_total ? v + load(grad_total + c) : v);
      if (part) part[c] = fmaf(load(grad_out + c), t * r, row == blockIdx.x ? 0.0f : part[c]);
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
  if (threadIdx.x % 32 == 0 && first + column < k) store(grad_weight + first + column, sum);
}

// Which way rows of k are moved: `rows` are the tensors and the values between their rows.
struct Rows {
  const void* at;
  int64_t stride;
};
template <typename T>
Way way_of(int64_t k, std::initializer_list<Rows> rows) {
  constexpr int kN = 16 / int(sizeof(T));
  bool whole = k % kN == 0, alike = k >= 8 * kN;
  for (const Rows& r : rows) {
    if (!r.at) continue;
    const bool on_boundary = reinterpret_cast<uintptr_t>(r.at) % 16 == 0;
    whole = whole && on_boundary && r.stride % kN == 0;
    alike = alike && on_boundary && r.stride % kN == k % kN;
  }
  return whole ? kWhole : alike ? kSkewed : kSingle;
}

template <int kTeam, int kCount>
struct Form {
  static constexpr int kThreads = kTeam, kVectors = kCount;
};
// Calls f with the way and the form for rows of k; false where none holds them.
template <typename T, typename F>
bool with_form(Way way, int64_t k, F&& f) {
  constexpr int kN = 16 / int(sizeof(T));
  const int64_t vectors = k / kN;
  // Threads that a row just fills, three or four vectors each: bytes on their way are what counts (rows of 1,288 bf16, 400 MB
  // in all, 61 us, by 128 threads with two vectors in some 86; of 1,041 81 and 153). Long ones with fewer vectors in more threads
  // are no quicker (8,193 bf16 67 us, by 1,024 threads 76), nor are more vectors in each than a row needs: 10,240 float32
  // 68 us with six, 99 with seven. Rows that do not fill what they take pay for it: 16,392 bf16 with six vectors 118 us (16,384
  // with four 74), 14,000 float32 with eight 85 (at a copy's rate 61).
  if (way == kWhole) {
    const auto g = [&](auto form) { return f(std::integral_constant<Way, kWhole>(), form), true; };
    if (vectors <= 8) return g(Form<8, 1>());
    if (vectors <= 16) return g(Form<16, 1>());
    if (vectors <= 32) return g(Form<32, 1>());
    if (vectors <= 64) return g(Form<32, 2>());
    if (vectors <= 96) return g(Form<32, 3>());
    if (vectors <= 128) return g(Form<32, 4>());
    if (vectors <= 192) return g(Form<64, 3>());
    if (vectors <= 256) return g(Form<64, 4>());
    if (vectors <= 384) return g(Form<128, 3>());
    if (vectors <= 512) return g(Form<128, 4>());
    if (vectors <= 768) return g(Form<256, 3>());
    if (vectors <= 1024) return g(Form<256, 4>());
    if (vectors <= 1536) return g(Form<512, 3>());
    if (vectors <= 2048) return g(Form<512, 4>());
    if (vectors <= 512 * 6) return g(Form<512, 6>());
    if (vectors <= 4096) return g(Form<512, 8>());
  } else if (way == kSkewed) {
    const auto g = [&](auto form) { return f(std::integral_constant<Way, kSkewed>(), form), true; };
    if (vectors <= 16) return g(Form<16, 1>());
    if (vectors <= 32) return g(Form<32, 1>());
    if (vectors <= 64) return g(Form<32, 2>());
    if (vectors <= 96) return g(Form<32, 3>());
    if (vectors <= 128) return g(Form<32, 4>());
    if (vectors <= 192) return g(Form<64, 3>());
    if (vectors <= 256) return g(Form<64, 4>());
    if (vectors <= 384) return g(Form<128, 3>());
    if (vectors <= 512) return g(Form<128, 4>());
    if (vectors <= 768) return g(Form<256, 3>());
    if (vectors <= 1024) return g(Form<256, 4>());
    if (vectors <= 1536) return g(Form<512, 3>());
    if (vectors <= 2048) return g(Form<512, 4>());
    if (vectors <= 512 * 6) return g(Form<512, 6>());
    if (vectors <= 4096) return g(Form<512, 8>());
  }
  const auto g = [&](auto form) { return f(std::integral_constant<Way, kSingle>(), form), true; };
  if (k <= 32) return g(Form<32, 1>());
  if (k <= 128) return g(Form<32, 4>());
  if (k <= 256) return g(Form<32, 8>());
  if (k <= 512) return g(Form<64, 8>());
  if (k <= 1024) return g(Form<128, 8>());
  if (k <= 4096) return g(Form<512, 8>());
  if (k <= 16384) return g(Form<1024, 16>());
  return false;
}
// The gradient holds three rows, the next three and the weight's gradient.
template <typename T, typename F>
bool with_grad_form(Way way, int64_t k, F&& f) {
  constexpr int kN = 16 / int(sizeof(T));
  const int64_t vectors = k / kN;
  if (way == kWhole) {
    const auto g = [&](auto form) { return f(std::integral_constant<Way, kWhole>(), form), true; };
    if (vectors <= 8) return g(Form<8, 1>());
    if (vectors <= 16) return g(Form<16, 1>());
    if (vectors <= 32) return g(Form<32, 1>());
    if (vectors <= 64) return g(Form<32, 2>());
    if (vectors <= 128) return g(Form<64, 2>());
    if (vectors <= 256) return g(Form<128, 2>());
    if (vectors <= 512) return g(Form<256, 2>());
    if (vectors <= 1024) return g(Form<512, 2>());
    if (vectors <= 2048) return g(Form<512, 4>());
    if constexpr (sizeof(T) == 4)
      if (vectors <= 4096) return g(Form<512, 8>());
  } else if (way == kSkewed) {
    const auto g = [&](auto form) { return f(std::integral_constant<Way, kSkewed>(), form), true; };
    if (vectors <= 32) return g(Form<32, 1>());
    if (vectors <= 64) return g(Form<32, 2>());
    if (vectors <= 128) return g(Form<64, 2>());
    if (vectors <= 256) return g(Form<128, 2>());
    if (vectors <= 512) return g(Form<256, 2>());
    if (vectors <= 1024) return g(Form<512, 2>());
    if (vectors <= 2048) return g(Form<512, 4>());
    if constexpr (sizeof(T) == 4)
      if (vectors <= 4096) return g(Form<512, 8>());
  }
  const auto g = [&](auto form) { return f(std::integral_constant<Way, kSingle>(), form), true; };
  if (k <= 32) return g(Form<32, 1>());
  if (k <= 128) return g(Form<32, 4>());
  if (k <= 256) return g(Form<32, 8>());
  if (k <= 512) return g(Form<64, 8>());
  if (k <= 1024) return g(Form<128, 8>());
  if (k <= 4096) return g(Form<512, 8>());
  if (k <= 8192) return g(Form<512, 16>());
  return false;
}

template <typename T, bool kCodes>
int norm(const Norm& p, cudaStream_t s) {
  // codes start on boundaries of a vector's values where whole rows do
  const Way way = way_of<T>(p.k, {{p.x, p.x_stride}, {p.residual, p.residual_stride}, {p.out, p.k}, {p.total, p.k}, {p.weight, p.k}});
  const bool held = with_form<T>(kCodes && way == kWhole && (reinterpret_cast<uintptr_t>(p.codes) | p.pitch) % 16 ? kSingle : way,
                                 p.k, [&](auto of_way, auto form) {
    using G = Team<form.kThreads>;
    norm_kernel<T, of_way.value, form.kThreads, form.kVectors, kCodes>
        <<<unsigned((p.m + G::kRows - 1) / G::kRows), G::kBlock, 0, s>>>(p);
  });
  if (!held) long_norm_kernel<T, kCodes><<<unsigned(p.m), kLong, 0, s>>>(p);
  return launch_status();
}

// Blocks of the gradient's kernel, each with a row of the weight's gradient in scratch: two an SM (128,000 x 512 bf16 87 us;
// one 114, three 106, four 95), of those that fill an SM one (1,000 x 16,384 bf16 49 us, two one after the other 62), and of few
// rows fewer, so that a team has some. Multiples of 8 where it has more than one.
constexpr int kGradBlocks = 2 * 148, kGradBlocksAlone = 144;
int64_t grad_blocks(int64_t rows, int64_t most) {
  return rows <= 144 ? rows : rows < 4 * 144 ? 144 : rows < 4 * most ? rows / 4 / 8 * 8 : most;
}

template <typename T>
int norm_grad(const NormGrad& p, void* grad_weight, cudaStream_t s) {
  const Way way = way_of<T>(p.k, {{p.grad_out, p.grad_out_stride}, {p.total, p.total_stride}, {p.grad_total, p.grad_total_stride},
                                  {p.grad, p.k}, {p.weight, p.k}});
  int64_t blocks = grad_blocks(p.m, kGradBlocks);
  cudaError_t shared_memory = cudaSuccess;
  const bool held = with_grad_form<T>(way, p.k, [&](auto of_way, auto form) {
    using G = Team<form.kThreads>;
    blocks = grad_blocks((p.m + G::kRows - 1) / G::kRows, G::kBlock > 256 ? kGradBlocksAlone : kGradBlocks);
    constexpr int kApart = Grads<T, of_way.value, form.kThreads, form.kVectors>::kApartBytes;
    // columns' sums of more rows than one, or a thread's own
    const size_t shared = kApart ? kApart : G::kRows > 1 ? p.k * sizeof(float) : 0;
    const auto kernel = norm_grad_kernel<T, of_way.value, form.kThreads, form.kVectors>;
    if constexpr (kApart > 0) shared_memory = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kApart);
    if (shared_memory == cudaSuccess) kernel<<<unsigned(blocks), G::kBlock, shared, s>>>(p);
  });
  if (shared_memory != cudaSuccess) return int(shared_memory);
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
  return (m < kGradBlocks ? m : kGradBlocks) * k * 4;
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
