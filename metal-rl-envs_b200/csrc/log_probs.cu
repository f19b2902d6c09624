// Scores of actions: the log-probability of a chosen one, the entropy and the best alternatives of rows of logits, and
// their gradient. With the largest logit b of a row (of those allowed; others count as -infinity),
//     S = sum e^(l - b),   W = sum e^(l - b) (l - b),   normalizer = b + log S,   entropy = log S - W / S,
// and sums over parts of a row join: (b, S, W) moves to a larger b' by d = b - b': (e^d S, e^d (W + S d)).
// The gradient: g ([j = action] - p_j) - h p_j (log p_j + entropy), p_j = e^(l_j - normalizer), the normalizer with what its
// rounding to a float32 has left (`remainder`): for b far from zero that is as large as log S.
//
// A row is read once: any number will do for b that is not far below the largest logit, so that sums begin with the first
// vectors and nothing waits for a largest one. The bound is memory, with the power unit close behind (a logit is one
// power, 16 a clock and SM, and some 8 instructions of which half work on two values): 4,096 x 32,768 bf16 49 us (5.5 TB/s),
// with eight alternatives 62, with a mask 70 (5.7 TB/s), 3,000 x 32,768 float32 66 (5.9 TB/s); the gradient
// of 4,096 x 16,384 bf16 48 us (5.6 TB/s), float32 85 (6.3 TB/s), of 4,096 x 32,771 bf16 with a mask 120 (5.6 TB/s). Other
// arrangements of the forward pass, for 4,096 x 32,768 bf16 with eight alternatives: a row in a block's registers, its largest
// logit first, 128 us (barriers); in its shared memory 126; a warp a row, alternatives kept as they come, 170 (insertions).
#include <cooperative_groups.h>
#include <cuda_bf16.h>

#include <type_traits>

#include "common.cuh"

namespace rlenv {
namespace {

namespace cg = cooperative_groups;

constexpr int kMostTop = 32;
constexpr float kFar = -200.0f;  // e^kFar is 0 in float32: what lies further below the largest logit adds nothing

RLENV_D float infinity() { return __uint_as_float(0x7f800000u); }
RLENV_D float not_a_number() { return __uint_as_float(0x7fffffffu); }
// The larger, or NaN where one is.
RLENV_D float larger(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

struct Scores {
  int64_t m, v;
  const void* logits;
  int64_t stride;
  const void* actions;
  int action_dtype;
  const uint8_t* allowed;  // null: all
  int64_t allowed_stride;
  float *log_prob, *entropy, *normalizer;
  int top;
  int64_t* top_actions;
  float* top_log_probs;
  float* remainder;  // of the normalizer; may be null
};

RLENV_D int64_t action_of(const void* actions, int dtype, int64_t row) {
  if (dtype == RLENV_I64) return __ldg(static_cast<const long long*>(actions) + row);
  if (dtype == RLENV_I32) return __ldg(static_cast<const int*>(actions) + row);
  return __ldg(static_cast<const unsigned char*>(actions) + row);
}

RLENV_D float value_at(const float* from) { return __ldg(from); }
RLENV_D float value_at(const __nv_bfloat16* from) {
  return __uint_as_float(uint32_t(__ldg(reinterpret_cast<const unsigned short*>(from))) << 16);
}

RLENV_D float exp2_fast(float x) {  // within 2 ulp, 0 where float32's normal numbers end
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
constexpr float kLog2E = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

// log2 e^(l - base) of two logits. What lies further below than kFar counts as that: it adds nothing, and -infinity times
// nothing would be NaN.
RLENV_D uint64_t powers_of(uint64_t l, uint64_t minus_base) {
  const float2 d = values_of(add_pairs(l, minus_base));
  return multiply_pairs(pair_of(larger(d.x, kFar), larger(d.y, kFar)), pair_of(kLog2E, kLog2E));
}

// Logits are ordered by value, ties by the lower place: as one whole number, larger first. 0 stands below all, NaN
// above.
RLENV_D uint32_t order_of(float x) {
  if (x != x) return 0xfffffffeu;  // so that no key is all ones
  const uint32_t b = x == 0.0f ? 0u : __float_as_uint(x);  // both zeros are one
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
RLENV_D float value_of(uint32_t order) {
  return __uint_as_float(order & 0x80000000u ? order & 0x7fffffffu : ~order);
}
RLENV_D uint64_t key_of(float x, uint32_t place) { return uint64_t(order_of(x)) << 32 | ~place; }

// Of a part of a row: its largest logit, and S and W against it (against 0 where that is -infinity: both are 0 then).
struct Sums {
  float m, s, w;
};
RLENV_D float base_of(float largest) { return largest == -infinity() ? 0.0f : largest; }
RLENV_D Sums moved(const Sums& a, float m) {  // against m >= a.m
  if (a.s == 0.0f) return {m, 0.0f, 0.0f};
  const float d = larger(a.m - m, kFar), e = __expf(d);
  return {m, e * a.s, e * fmaf(a.s, d, a.w)};
}
// The largest of kLanes neighbouring lanes', or NaN, known to all of them.
template <int kLanes>
RLENV_D float largest_of_lanes_of(float x) {
  if constexpr (kLanes == 32) {
    float r;
    asm volatile("redux.sync.max.NaN.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(x));
    return r;
  } else {
#pragma unroll
    for (int d = kLanes / 2; d > 0; d /= 2) x = larger(x, __shfl_xor_sync(0xffffffffu, x, d));
    return x;
  }
}
// Of kLanes neighbouring lanes, known to all of them.
template <int kLanes>
RLENV_D Sums of_team(const Sums& a) {
  const Sums own = moved(a, largest_of_lanes_of<kLanes>(a.m));
  uint64_t both = pair_of(own.s, own.w);
#pragma unroll
  for (int d = kLanes / 2; d > 0; d /= 2) both = add_pairs(both, __shfl_xor_sync(0xffffffffu, both, d));
  const float2 of = values_of(both);
  return {own.m, of.x, of.y};
}
// A row's normalizer as the two terms that it is the sum of: subtracted from a logit one after the other they leave a
// log-probability whose error does not grow with what the row's logits have in common (eight equal logits of 1e5: -2.0794415, less
// the rounded sum -2.078125).
struct Normalizer {
  float base, log_sum;
  bool none;  // a row that allows nothing: its normalizer is -infinity, and so is a logit less either term
  RLENV_D explicit Normalizer(const Sums& a) : base(base_of(a.m)), log_sum(a.s == 0.0f ? 0.0f : logf(a.s)), none(a.s == 0.0f) {}
  RLENV_D float whole() const { return none ? -infinity() : base + log_sum; }
  RLENV_D float remainder() const {  // exactly what whole() leaves (Knuth's two-sum)
    const float n = whole(), b = n - base;
    return fabsf(n) < infinity() ? (base - (n - b)) + (log_sum - b) : 0.0f;
  }
  RLENV_D float log_prob(float l) const { return (l - base) - log_sum; }
};

// A row's action and its logit, read before the row so that nothing waits for them after it.
struct Chosen {
  int64_t action;
  float l;
  template <typename T>
  static RLENV_D Chosen of(const Scores& p, int64_t row, const T* logits, const uint8_t* allowed) {
    const int64_t a = action_of(p.actions, p.action_dtype, row);
    return {a, a >= 0 && a < p.v && (!allowed || allowed[a]) ? value_at(logits + a) : -infinity()};
  }
};

RLENV_D void write_scores(const Scores& p, int64_t row, const Sums& sums, const Normalizer& normalizer, const Chosen& chosen) {
  p.normalizer[row] = normalizer.whole();
  if (p.remainder) p.remainder[row] = normalizer.remainder();
  p.entropy[row] = normalizer.none ? 0.0f : normalizer.log_sum - sums.w / sums.s;
  check_flag(chosen.action >= p.v, kCheckActionRange);
  p.log_prob[row] = chosen.action < 0 ? 0.0f : chosen.action >= p.v ? not_a_number() : normalizer.log_prob(chosen.l);
}
RLENV_D void write_top(const Scores& p, int64_t row, int rank, uint64_t key, const Normalizer& normalizer) {
  p.top_actions[row * p.top + rank] = int64_t(uint32_t(~uint32_t(key)));
  p.top_log_probs[row * p.top + rank] = normalizer.log_prob(value_of(uint32_t(key >> 32)));
}

// ---- few actions: a row is the work of kLanes neighbouring lanes, kEach logits of it in each --------------
//
// Rows of up to 1,024 lie in registers whole. What a row costs is instructions: half of them its logits, half its end (joins,
// logarithms, the action), which many logits a lane and few lanes a row make cheaper (169,089 of 200 float32 by 16 lanes 32 us,
// by 32 43; 131,072 of 1,000 bf16 93 us, of 500 51; as long rows are taken, below, 102 and 112).

// A key of a logit among up to 128, larger first, each another; 0 is none. bfloat16 orders leave 16 bits for the place.
RLENV_D uint64_t few_key(const float*, float x, int place) { return key_of(x, place); }
RLENV_D uint32_t few_key(const __nv_bfloat16*, float x, int place) { return (order_of(x) & 0xffff0000u) | (0xffffu - place); }
RLENV_D uint64_t whole_key(uint64_t key) { return key; }
RLENV_D uint64_t whole_key(uint32_t key) {
  const uint32_t order = key & 0x80000000u ? key & 0xffff0000u : key | 0xffffu;
  return uint64_t(order) << 32 | (key | 0xffff0000u);
}
template <int kLanes, typename K>
RLENV_D K largest_of_team(K key) {
  if constexpr (kLanes == 32) {
    const uint32_t high = __reduce_max_sync(0xffffffffu, uint32_t(key >> 32));
    return K(high) << 32 | __reduce_max_sync(0xffffffffu, uint32_t(key >> 32) == high ? uint32_t(key) : 0u);
  } else {
#pragma unroll
    for (int d = kLanes / 2; d > 0; d /= 2) {
      const K other = __shfl_xor_sync(0xffffffffu, key, d);
      key = other > key ? other : key;
    }
    return key;
  }
}
// The row's best `top` logits, one after the other: each lane's own are sorted, and the lane whose first is the row's best gives
// it up. The lanes write together, each kLanes-th of them. A search through all lanes' logits for each takes twice as long
// (192,341 of 41 float32 with twenty alternatives 90 us, by searches 187; 169,089 of 100 bf16 with eight 59 and 314).
template <typename T, int kLanes, int kEach>
RLENV_D void few_best(const Scores& p, int64_t row, bool real, int sub, const float (&x)[kEach], const Normalizer& normalizer) {
  using K = decltype(few_key(static_cast<const T*>(nullptr), 0.0f, 0));
  K keys[kEach];
#pragma unroll
  for (int i = 0; i < kEach; ++i) {
    const int j = sub + kLanes * i;
    keys[i] = j < p.v ? few_key(static_cast<const T*>(nullptr), x[i], j) : K(0);
  }
  const auto order = [&](int i, int j) {
    const K high = keys[i] > keys[j] ? keys[i] : keys[j], low = keys[i] > keys[j] ? keys[j] : keys[i];
    keys[i] = high, keys[j] = low;
  };
  if (p.top == 1) {
#pragma unroll
    for (int d = kEach / 2; d > 0; d /= 2)
#pragma unroll
      for (int i = 0; i < d; ++i) order(i, i + d);
  } else {  // odd-even merges
#pragma unroll
    for (int n = 1; n < kEach; n *= 2)
#pragma unroll
      for (int d = n; d > 0; d /= 2)
#pragma unroll
        for (int i = 0; i + d < kEach; ++i)
          if (i >= d % n && (i - d % n) / d % 2 == 0 && i / (2 * n) == (i + d) / (2 * n)) order(i, i + d);
  }
  K mine = 0;
  for (int r = 0; r < p.top; ++r) {
    const K best = largest_of_team<kLanes>(keys[0]);
    const bool own = keys[0] == best;
#pragma unroll
    for (int i = 0; i < kEach - 1; ++i) keys[i] = own ? keys[i + 1] : keys[i];
    keys[kEach - 1] = own ? K(0) : keys[kEach - 1];
    if (r % kLanes == sub) mine = best;
    if ((r % kLanes == kLanes - 1 || r == p.top - 1) && real && sub <= r % kLanes)
      write_top(p, row, r - r % kLanes + sub, whole_key(mine), normalizer);
  }
}

// The same where a warp has a row: as many lanes as alternatives are asked for have a logit that reaches the top-th of the
// lanes' largest, and the logits that do, few more than `top`, are ranked by counting (169,089 of 200 float32 with eight
// alternatives 98 us, by sorting 206; 131,072 of 500 bf16 with twenty 149).
constexpr int kFound = 64;
struct Found {
  uint64_t keys[kFound];
  int count;
};
template <typename T, int kEach>
RLENV_D void few_best_of_warp(const Scores& p, int64_t row, const float (&x)[kEach], const Normalizer& normalizer, Found& found) {
  const int lane = threadIdx.x % 32, left = int(p.v) - lane;
  float most = x[0];
#pragma unroll
  for (int i = 1; i < kEach; ++i) most = larger(most, x[i]);
  if (lane == 0) found.count = 0;
  __syncwarp();
  uint32_t order = left > 0 ? order_of(most) : 0, least = 0;
  for (int r = 0; r < p.top; ++r) {
    least = __reduce_max_sync(0xffffffffu, order);
    if (lane == __ffs(__ballot_sync(0xffffffffu, order == least)) - 1) order = 0;
  }
  const float bar = value_of(least);
  uint32_t reach = 0;
#pragma unroll
  for (int i = 0; i < kEach; ++i)
    if (32 * i < left && !(x[i] < bar)) reach |= 1u << i;
  if (reach) {
    const T* const logits = static_cast<const T*>(p.logits) + row * p.stride;
    const uint8_t* const allowed = p.allowed ? p.allowed + row * p.allowed_stride : nullptr;
    int at = atomicAdd(&found.count, __popc(reach));
    for (; reach && at < kFound; reach &= reach - 1, ++at) {
      const int j = lane + 32 * (__ffs(reach) - 1);
      found.keys[at] = key_of(allowed && !allowed[j] ? -infinity() : value_at(logits + j), j);
    }
  }
  __syncwarp();
  const int count = found.count;
  if (count <= kFound) {
    for (int i = lane; i < count; i += 32) {
      const uint64_t key = found.keys[i];
      int above = 0;
#pragma unroll 4
      for (int k = 0; k < count; ++k) above += found.keys[k] > key;
      if (above < p.top) write_top(p, row, above, key, normalizer);
    }
  } else {  // equal ones: the largest is taken out, one after the other
    uint64_t last = ~uint64_t(0);
    for (int r = 0; r < p.top; ++r) {
      uint64_t own = 0;
#pragma unroll
      for (int i = 0; i < kEach; ++i) {
        const uint64_t key = 32 * i < left ? key_of(x[i], lane + 32 * i) : 0;
        if (key < last && key > own) own = key;
      }
      last = largest_of_team<32>(own);
      if (lane == 0) write_top(p, row, r, last, normalizer);
    }
  }
}

// Loads where there is a place, as single instructions: branches around loads would have each wait for the one before.
RLENV_D void load_if(int there, const float* from, float& to) {
  asm volatile("{\n\t.reg .pred in;\n\tsetp.gt.s32 in, %2, 0;\n\t@in ld.global.nc.f32 %0, [%1];\n\t}" : "+f"(to) : "l"(from), "r"(there));
}
RLENV_D void load_if(int there, const __nv_bfloat16* from, uint16_t& to) {
  asm volatile("{\n\t.reg .pred in;\n\tsetp.gt.s32 in, %2, 0;\n\t@in ld.global.nc.u16 %0, [%1];\n\t}" : "+h"(to) : "l"(from), "r"(there));
}
RLENV_D void load_if(int there, const uint8_t* from, uint16_t& to) {
  asm volatile("{\n\t.reg .pred in;\n\tsetp.gt.s32 in, %2, 0;\n\t@in ld.global.nc.u8 %0, [%1];\n\t}" : "+h"(to) : "l"(from), "r"(there));
}
RLENV_D float value_in(float x) { return x; }
RLENV_D float value_in(uint16_t bits) { return __uint_as_float(uint32_t(bits) << 16); }
// A lane's logits of a row: places sub, sub + kLanes and so on.
template <int kLanes, int kEach, typename T, typename P>
RLENV_D void few_logits(const P& p, int64_t row, int sub, float (&x)[kEach]) {
  using Raw = std::conditional_t<sizeof(T) == 4, float, uint16_t>;
  const T* const logits = static_cast<const T*>(p.logits) + row * p.stride + sub;
  const uint8_t* const allowed = p.allowed + row * p.allowed_stride + sub;
  const int left = int(p.v) - sub;
  Raw raw[kEach];
  uint16_t open[kEach];
#pragma unroll
  for (int i = 0; i < kEach; ++i) {
    if constexpr (sizeof(T) == 4)
      raw[i] = -infinity();
    else
      raw[i] = 0xff80;
    load_if(left - kLanes * i, logits + kLanes * i, raw[i]);
  }
  if (p.allowed) {
#pragma unroll
    for (int i = 0; i < kEach; ++i) open[i] = 1, load_if(left - kLanes * i, allowed + kLanes * i, open[i]);
#pragma unroll
    for (int i = 0; i < kEach; ++i) x[i] = open[i] == 0 ? -infinity() : value_in(raw[i]);
  } else {
#pragma unroll
    for (int i = 0; i < kEach; ++i) x[i] = value_in(raw[i]);
  }
}

// Three blocks an SM of lanes with 32 logits each, which the compiler by itself gives the registers of two (131,072 of 1,000
// bf16 94 us, else 126); for fewer logits it is left to itself (0).
template <typename T, int kLanes, int kEach>
__global__ void __launch_bounds__(256, kEach == 32 ? 3 : 0) few_scores_kernel(const __grid_constant__ Scores p) {
  const int sub = threadIdx.x % kLanes;
  const int64_t at = (int64_t(blockIdx.x) * 256 + threadIdx.x) / kLanes, row = at < p.m ? at : p.m - 1;
  float x[kEach];
  few_logits<kLanes, kEach, T>(p, row, sub, x);
  const Chosen chosen = Chosen::of(p, row, static_cast<const T*>(p.logits) + row * p.stride,
                                   p.allowed ? p.allowed + row * p.allowed_stride : nullptr);
  Sums sums{x[0], 0.0f, 0.0f};
#pragma unroll
  for (int i = 1; i < kEach; ++i) sums.m = larger(sums.m, x[i]);
  sums.m = largest_of_lanes_of<kLanes>(sums.m);
  const float base = base_of(sums.m);
  const uint64_t minus_base = pair_of(-base, -base);
  uint64_t s2 = 0, w2 = 0;
#pragma unroll
  for (int i = 0; i < kEach; i += 2) {
    const uint64_t y = powers_of(pair_of(x[i], x[i + 1]), minus_base);
    const float2 of = values_of(y);
    const uint64_t e = pair_of(exp2_fast(of.x), exp2_fast(of.y));
    s2 = add_pairs(s2, e), w2 = multiply_add_pairs(e, y, w2);
  }
  const float2 s_own = values_of(s2), w_own = values_of(w2);
  uint64_t both = pair_of(s_own.x + s_own.y, (w_own.x + w_own.y) * kLn2);
#pragma unroll
  for (int d = kLanes / 2; d > 0; d /= 2) both = add_pairs(both, __shfl_xor_sync(0xffffffffu, both, d));
  const float2 of = values_of(both);
  sums.s = of.x, sums.w = of.y;
  const Normalizer normalizer(sums);
  if (sub == 0 && at < p.m) write_scores(p, row, sums, normalizer, chosen);
  if constexpr (kLanes == 32) {
    __shared__ Found found[8];
    if (p.top > 0 && at < p.m) few_best_of_warp<T, kEach>(p, row, x, normalizer, found[threadIdx.x / 32]);
  } else if constexpr (kLanes < 16) {
    if (p.top > 0) few_best<T, kLanes, kEach>(p, row, at < p.m, sub, x, normalizer);
  }
}

// ---- more: a row is the work of a warp, a block or a cluster of blocks -----------------------------------

// A row's logits as 16-byte vectors from the last boundary before its first: vector i holds the places from
// i kValues - skip on.
template <typename T>
struct Grid {
  static constexpr int kValues = 16 / int(sizeof(T));
  const T* row;
  int64_t v;
  int skip;
  RLENV_D Grid(const T* row, int64_t v)
      : row(row), v(v), skip(int(reinterpret_cast<uintptr_t>(row) % 16 / sizeof(T))) {}
  RLENV_D int64_t vectors() const { return (v + skip + kValues - 1) / kValues; }
  RLENV_D int64_t place(int64_t i) const { return i * kValues - skip; }
};

// A vector is four words of 32 bits, each one float32 or two bfloat16 logits.
template <typename T>
RLENV_D float word_value(const uint32_t (&w)[4], int j) {
  if constexpr (sizeof(T) == 4)
    return __uint_as_float(w[j]);
  else
    return __uint_as_float(j % 2 ? w[j / 2] & 0xffff0000u : w[j / 2] << 16);
}
template <typename T>
RLENV_D uint64_t word_pair(const uint32_t (&w)[4], int i) {  // values 2 i and 2 i + 1
  return pair_of(word_value<T>(w, 2 * i), word_value<T>(w, 2 * i + 1));
}
RLENV_D __nv_bfloat162 as_bf162(uint32_t w) { return *reinterpret_cast<const __nv_bfloat162*>(&w); }
template <typename T>
RLENV_D uint32_t larger_words(uint32_t a, uint32_t b) {  // place by place, or NaN
  if constexpr (sizeof(T) == 4) return __float_as_uint(larger(__uint_as_float(a), __uint_as_float(b)));
  const __nv_bfloat162 p = __hmax2_nan(as_bf162(a), as_bf162(b));
  return *reinterpret_cast<const uint32_t*>(&p);
}
template <typename T>
RLENV_D float largest_of(uint32_t w) {
  if constexpr (sizeof(T) == 4) return __uint_as_float(w);
  return larger(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}
template <typename T>
RLENV_D constexpr uint32_t empty_word() {  // -infinity
  return sizeof(T) == 4 ? 0xff800000u : 0xff80ff80u;
}

// The kValues bytes of `allowed` from place j0 on, all of them in the row of v, as words.
template <int kValues>
RLENV_D uint2 bytes_at(const uint8_t* allowed, int64_t j0, int64_t v) {
  const uint8_t* const at = allowed + j0;
  const unsigned off = unsigned(reinterpret_cast<uintptr_t>(at) % kValues);
  uint2 b = make_uint2(0, 0);
  if (off == 0) {
    if constexpr (kValues == 8)
      b = __ldg(reinterpret_cast<const uint2*>(at));
    else
      b.x = __ldg(reinterpret_cast<const uint32_t*>(at));
  } else if (j0 >= 4 && j0 + kValues + 4 <= v) {  // the words around them are in the row too
    const uint32_t* const words = reinterpret_cast<const uint32_t*>(at - off % 4);
    const uint32_t w1 = __ldg(words + 1);
    b.x = __funnelshift_r(__ldg(words), w1, 8 * (off % 4));
    if (kValues == 8) b.y = __funnelshift_r(w1, off % 4 ? __ldg(words + 2) : 0u, 8 * (off % 4));
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      b.x |= uint32_t(at[i]) << 8 * i;
      if (kValues == 8) b.y |= uint32_t(at[4 + i]) << 8 * i;
    }
  }
  return b;
}
// kValues logits from place j0 on, which need not be a boundary; the places before and after them are in the row too.
template <typename T>
RLENV_D uint4 words_between(const T* row, int64_t j0) {
  const T* const at = row + j0;
  const bool between = sizeof(T) == 2 && reinterpret_cast<uintptr_t>(at) % 4;
  const uint32_t* const words = reinterpret_cast<const uint32_t*>(between ? at - 1 : at);
  uint32_t w[5];
#pragma unroll
  for (int i = 0; i < 4; ++i) w[i] = __ldg(words + i);
  if (!between) return make_uint4(w[0], w[1], w[2], w[3]);
  w[4] = __ldg(words + 4);
  return make_uint4(__funnelshift_r(w[0], w[1], 16), __funnelshift_r(w[1], w[2], 16), __funnelshift_r(w[2], w[3], 16),
                    __funnelshift_r(w[3], w[4], 16));
}
// Bytes that hold bit 7 of a byte of x eight times over: of byte n where the selector's digit is 8 + n.
RLENV_D uint32_t repeat_signs(uint32_t x, uint32_t selector) {
  uint32_t r;
  asm("prmt.b32 %0, %1, 0, %2;" : "=r"(r) : "r"(x), "r"(selector));
  return r;
}
// A vector's words with -infinity in the places whose bytes are zero.
template <typename T>
RLENV_D void cut_out(uint32_t (&w)[4], uint2 bytes) {
  // bit 7 of each byte that is not zero, then all bits of the values' places
  const auto marked = [](uint32_t b) { return (((b & 0x7f7f7f7fu) + 0x7f7f7f7fu) | b) & 0x80808080u; };
  const uint32_t of[2] = {marked(bytes.x), marked(bytes.y)};
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const uint32_t open = Grid<T>::kValues == 8 ? repeat_signs(of[k / 2], k % 2 ? 0xbbaa : 0x9988)
                                                : repeat_signs(of[0], 0x8888 + 0x1111 * k);
    w[k] = (w[k] & open) | (empty_word<T>() & ~open);
  }
}
// A vector that a row's end cuts: -infinity where a place is not in the row or not allowed. All loads go out before any is
// looked at.
template <typename T>
__device__ __noinline__ uint4 edge_vector(const T* row, const uint8_t* allowed, int64_t v, int64_t j0) {
  constexpr int kValues = 16 / int(sizeof(T));
  float x[kValues];
  uint8_t open[kValues];
#pragma unroll
  for (int j = 0; j < kValues; ++j) {
    const bool in = j0 + j >= 0 && j0 + j < v;
    x[j] = -infinity(), open[j] = 1;
    if (in) x[j] = value_at(row + j0 + j);
    if (in && allowed) open[j] = __ldg(allowed + j0 + j);
  }
  uint32_t w[4] = {0, 0, 0, 0};
#pragma unroll
  for (int j = 0; j < kValues; ++j) {
    const uint32_t bits = open[j] ? __float_as_uint(x[j]) : 0xff800000u;
    if constexpr (sizeof(T) == 4)
      w[j] = bits;
    else
      w[j / 2] |= bits >> 16 << 16 * (j % 2);
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// A warp's search for its best logits. Its part of a row is 32 lanes' vectors of up to kEpochs epochs, each of which leaves
// its largest logit behind. The top-th largest of a warp's (of several warps: of their lanes') has `top` logits at least that
// are not below it, and the groups which reach it, `top` of them where none are equal, are looked through again.
constexpr int kEpochs = 4;
struct Best {
  static constexpr int kMany = 64, kRoom = kMany + 256;  // a step adds one vector a lane, 256 logits at most
  uint64_t* keys;  // kRoom
  union {
    uint32_t largest[kEpochs][32];  // orders; 0: none. Until the groups are chosen
    struct {
      uint64_t kept[kMostTop];
      uint8_t groups[32 * kEpochs];
    };
  };
  int count;
  RLENV_D void add(uint64_t key) { keys[atomicAdd(&count, 1)] = key; }
  // Keeps the best `top` keys, in order. The smallest of them, or 0 where there are fewer. For the whole warp. Few are
  // ranked by counting, of many (a row of equal logits) the largest is taken out, one after the other.
  RLENV_D uint64_t keep(int top) {
    __syncwarp();
    const int lane = threadIdx.x % 32, n = count;
    if (n <= kMany + 32) {
      for (int i = lane; i < n; i += 32) {
        const uint64_t key = keys[i];
        int above = 0;
#pragma unroll 4
        for (int k = 0; k < n; ++k) above += keys[k] > key;
        if (above < top) kept[above] = key;
      }
    } else {
      uint64_t last = ~uint64_t(0);
      for (int r = 0; r < top; ++r) {
        uint64_t own = 0;
        for (int i = lane; i < n; i += 32) {
          const uint64_t key = keys[i];
          if (key < last && key > own) own = key;
        }
        const uint32_t high = __reduce_max_sync(0xffffffffu, uint32_t(own >> 32)),
                       low = __reduce_max_sync(0xffffffffu, uint32_t(own >> 32) == high ? uint32_t(own) : 0u);
        last = uint64_t(high) << 32 | low;
        if (lane == 0) kept[r] = last;
      }
    }
    __syncwarp();
    if (lane < top && lane < n) keys[lane] = kept[lane];
    if (lane == 0) count = n < top ? n : top;
    const uint64_t least = n < top ? 0 : kept[top - 1];
    __syncwarp();
    return least;
  }
  // Lists the groups whose largest logit is not below `least`; returns their number.
  RLENV_D int list(int epochs, uint32_t least) {
    const int lane = threadIdx.x % 32;
    uint32_t of[kEpochs];
#pragma unroll
    for (int e = 0; e < kEpochs; ++e) of[e] = e < epochs ? largest[e][lane] : 0;
    __syncwarp();  // the list takes their place
    int n = 0;
#pragma unroll
    for (int e = 0; e < kEpochs; ++e) {
      const bool in = of[e] != 0 && of[e] >= least;
      const uint32_t all = __ballot_sync(0xffffffffu, in);
      if (in) groups[n + __popc(all & ((1u << lane) - 1))] = uint8_t(32 * e + lane);
      n += __popc(all);
    }
    __syncwarp();
    return n;
  }
};
// The n-th largest of a warp's whole numbers, four a lane: the largest is taken out, one after the other.
RLENV_D uint32_t nth_largest(uint32_t (&v)[4], int n) {
  const int lane = threadIdx.x % 32;
  const auto order = [&](int i, int j) {
    const uint32_t high = max(v[i], v[j]);
    v[j] = min(v[i], v[j]), v[i] = high;
  };
  order(0, 1), order(2, 3), order(0, 2), order(1, 3), order(1, 2);
  uint32_t largest = 0;
  for (int r = 0; r < n; ++r) {
    largest = __reduce_max_sync(0xffffffffu, v[0]);
    if (lane == __ffs(__ballot_sync(0xffffffffu, v[0] == largest)) - 1) v[0] = v[1], v[1] = v[2], v[2] = v[3], v[3] = 0;
  }
  return largest;
}

// kWarps warps read a row in turns of kSteps vectors a lane, and a cluster's blocks a part of it each: no lane waits for
// another before the row's end. Each lane's next turns are on their way into its own places of shared memory meanwhile. A
// lane's sums stand against a base of its own, which moves only where a logit is kAbove above it. log S and W / S have what the
// base lies below the largest logit in common and are rounded with it, so that it stays small: at 20 the entropy of rows whose
// largest logit comes late is off by up to 8e-6, at 3 by 4e-7, as rows that take the largest first (4,096 x 32,768 bf16 of
// deviation 2, 48.7 us at 20, 49.2 at 3).
constexpr int kSteps = 4, kAhead = 3;  // kAhead: turns in shared memory, the one at work among them
constexpr float kAbove = 3.0f;
template <int kWarps>
struct Team {
  static constexpr int kThreads = kWarps == 1 ? 128 : 32 * kWarps, kRows = kThreads / (32 * kWarps);
  static constexpr int kRing = kAhead * kSteps * 32;  // vectors of a warp
  static constexpr int kShared = kThreads / 32 * kRing * 16;
  static constexpr int kBlocks = 896 / kThreads < 2 ? 2 : 896 / kThreads;  // an SM's: what shared memory holds
};
static_assert(Team<1>::kRing * 16 >= Best::kRoom * 8, "the keys lie in the ring's place");

template <typename T, int kWarps>
__global__ void __launch_bounds__(Team<kWarps>::kThreads, Team<kWarps>::kBlocks)
scores_kernel(const __grid_constant__ Scores p) {
  using G = Team<kWarps>;
  constexpr int kValues = Grid<T>::kValues, kStride = 32 * kWarps, kTurn = kSteps * kStride, kBlockWarps = G::kThreads / 32;
  extern __shared__ __align__(16) uint4 rings[];
  __shared__ Best bests[kBlockWarps];
  __shared__ Sums of_warps[kBlockWarps];
  __shared__ Sums of_block;
  __shared__ uint64_t top_of_block[kMostTop];
  __shared__ uint32_t largest_of_lanes[kWarps == 1 ? 1 : 32 * kWarps];
  cg::cluster_group cluster = cg::this_cluster();
  const int blocks = kWarps == 16 ? int(cluster.num_blocks()) : 1, rank = blocks > 1 ? int(cluster.block_rank()) : 0;
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32 % kWarps;
  const int64_t row = kWarps == 1 ? int64_t(blockIdx.x) * kBlockWarps + threadIdx.x / 32 : blockIdx.x / blocks;
  if (row >= p.m) return;  // a warp
  const Grid<T> grid(static_cast<const T*>(p.logits) + row * p.stride, p.v);
  const uint8_t* const allowed = p.allowed ? p.allowed + row * p.allowed_stride : nullptr;
  const int vectors = int(grid.vectors()), part = (vectors + blocks - 1) / blocks, begin = min(rank * part, vectors),
            end = min(begin + part, vectors);
  // The row's first and last vectors, where they are not whole.
  const int first_whole = grid.skip > 0, last_whole = min((grid.skip + p.v) % kValues ? vectors - 1 : vectors, end);
  const auto whole = [&](int i) { return i >= first_whole && i < last_whole; };
  Best& best = bests[threadIdx.x / 32];
  uint4* const ring = rings + threadIdx.x / 32 * G::kRing;
  const int warp_begin = begin + 32 * warp, turns = warp_begin < end ? (end - warp_begin + kTurn - 1) / kTurn : 0;

  const auto largest_word = [](const uint32_t (&w)[4]) {
    return larger_words<T>(larger_words<T>(w[0], w[1]), larger_words<T>(w[2], w[3]));
  };
  const auto words = [](uint4 q, uint32_t (&w)[4]) { w[0] = q.x, w[1] = q.y, w[2] = q.z, w[3] = q.w; };
  const auto issue = [&](int turn, int slot) {
    if (turn < turns) {
      const int from = warp_begin + turn * kTurn, first = from + lane;
      uint4* const to = ring + slot * (kSteps * 32) + lane;
      const uint32_t to_at = uint32_t(__cvta_generic_to_shared(to));
      const T* const at = grid.row + grid.place(first);
      if (from >= first_whole && from + kTurn - kStride + 32 <= last_whole) {  // nothing but whole vectors
#pragma unroll
        for (int u = 0; u < kSteps; ++u)
          asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to_at + u * 512), "l"(at + u * kStride * kValues) : "memory");
      } else {
#pragma unroll 1
        for (int u = 0; u < kSteps; ++u) {
          const int i = first + u * kStride;
          if (whole(i))
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to_at + u * 512), "l"(at + u * kStride * kValues) : "memory");
          else if (i < end)
            to[u * 32] = edge_vector(grid.row, allowed, p.v, grid.place(i));
          else
            to[u * 32] = make_uint4(empty_word<T>(), empty_word<T>(), empty_word<T>(), empty_word<T>());
        }
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  uint2 bytes[kSteps];  // of the turn at work, read a turn ahead
  const auto load_bytes = [&](int turn) {
    const int from = warp_begin + turn * kTurn + lane;
#pragma unroll
    for (int u = 0; u < kSteps; ++u) {
      bytes[u] = make_uint2(~0u, ~0u);
      if (turn < turns && whole(from + u * kStride)) bytes[u] = bytes_at<kValues>(allowed, grid.place(from + u * kStride), p.v);
    }
  };

  float base = -infinity(), of_epoch = -infinity();
  uint64_t s2 = 0, w2 = 0;
  const auto own_sums = [&] {
    const float2 s = values_of(s2), w = values_of(w2);
    return Sums{base, s.x + s.y, (w.x + w.y) * kLn2};
  };
  // An epoch's turns, a power of two.
  const int epoch_bits = turns <= kEpochs ? 0 : 32 - __clz((turns - 1) / kEpochs), epoch = 1 << epoch_bits;
#pragma unroll
  for (int t = 0; t < kAhead - 1; ++t) issue(t, t);
  if (allowed) load_bytes(0);
  const Chosen chosen = Chosen::of(p, row, grid.row, allowed);
  int slot = 0, next = kAhead - 1, left = epoch, at_epoch = 0;
  for (int turn = 0; turn < turns; ++turn) {
    const int from = warp_begin + turn * kTurn;
    issue(turn + kAhead - 1, next);
    next = next == kAhead - 1 ? 0 : next + 1;
    asm volatile("cp.async.wait_group %0;" ::"n"(kAhead - 1) : "memory");
    uint32_t w[kSteps][4];
#pragma unroll
    for (int u = 0; u < kSteps; ++u) words(ring[(slot * kSteps + u) * 32 + lane], w[u]);
    slot = slot == kAhead - 1 ? 0 : slot + 1;
    if (allowed) {
#pragma unroll
      for (int u = 0; u < kSteps; ++u) cut_out<T>(w[u], bytes[u]);
      load_bytes(turn + 1);
    }
    uint32_t all = largest_word(w[0]);
#pragma unroll
    for (int u = 1; u < kSteps; ++u) all = larger_words<T>(all, largest_word(w[u]));
    const float most = largest_of<T>(all);
    if (most > base + kAbove) {
      const float d = larger(base - most, kFar) * kLog2E, e = exp2_fast(d);
      w2 = multiply_pairs(pair_of(e, e), multiply_add_pairs(s2, pair_of(d, d), w2)), s2 = multiply_pairs(pair_of(e, e), s2);
      base = most;
    }
    const float against = base_of(base);
    const uint64_t minus_base = pair_of(-against, -against);
#pragma unroll
    for (int u = 0; u < kSteps; ++u) {
      if (from + u * kStride >= end) break;
#pragma unroll
      for (int i = 0; i < kValues / 2; ++i) {
        const uint64_t y = powers_of(word_pair<T>(w[u], i), minus_base);
        const float2 of = values_of(y);
        const uint64_t e = pair_of(exp2_fast(of.x), exp2_fast(of.y));
        s2 = add_pairs(s2, e), w2 = multiply_add_pairs(e, y, w2);
      }
    }
    if (p.top > 0) {
      of_epoch = larger(of_epoch, most);
      if (--left == 0 || turn == turns - 1) {
        best.largest[at_epoch][lane] = warp_begin + at_epoch * epoch * kTurn + lane < end ? order_of(of_epoch) : 0;
        of_epoch = -infinity(), left = epoch, ++at_epoch;
      }
    }
  }
  Sums sums = of_team<32>(own_sums());

  if (p.top > 0) {
    if (lane == 0) best.count = 0, best.keys = reinterpret_cast<uint64_t*>(ring);
    __syncwarp();
    uint32_t of[kEpochs];
    static_assert(kEpochs == 4, "as nth_largest takes them");
#pragma unroll
    for (int e = 0; e < kEpochs; ++e) of[e] = e < at_epoch ? best.largest[e][lane] : 0;
    if constexpr (kWarps > 1) {
      largest_of_lanes[threadIdx.x] = max(max(of[0], of[1]), max(of[2], of[3]));
      __syncthreads();
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        of[e] = 0;
#pragma unroll
        for (int i = 0; i < kWarps / 4; ++i) of[e] = max(of[e], largest_of_lanes[32 * (e * (kWarps / 4) + i) + lane]);
      }
    }
    const uint32_t least = nth_largest(of, p.top);
    const int each_bits = 2 + epoch_bits, total = best.list(at_epoch, least) << each_bits;
    static_assert(kSteps == 4, "a group's vectors are 4 a turn");
    uint64_t least_key = uint64_t(least) << 32;
    const auto look_at = [&](int i, const uint32_t (&w)[4]) {  // vector i, for the whole warp
      const float bar = value_of(uint32_t(least_key >> 32));
      if (i < end && !(largest_of<T>(largest_word(w)) < bar)) {
        uint32_t reach = 0;
#pragma unroll
        for (int j = 0; j < kValues; ++j) reach |= !(word_value<T>(w, j) < bar) ? 1u << j : 0u;
        const int place0 = int(grid.place(i));
        for (; reach; reach &= reach - 1) {
          const int j = __ffs(reach) - 1, place = place0 + j;
          const uint32_t word = kValues == 4 ? (j < 2 ? (j < 1 ? w[0] : w[1]) : (j < 3 ? w[2] : w[3]))
                                             : (j < 4 ? (j < 2 ? w[0] : w[1]) : (j < 6 ? w[2] : w[3]));
          const float x = __uint_as_float(kValues == 4 ? word : j % 2 ? word & 0xffff0000u : word << 16);
          const uint64_t key = key_of(x, uint32_t(place));
          if (key > least_key && place >= 0 && place < p.v) best.add(key);
        }
      }
      __syncwarp();
      const int count = best.count;
      __syncwarp();  // all lanes have read it before one adds to it again: they keep together or not at all
      if (count > Best::kMany)
        if (const uint64_t now = best.keep(p.top)) least_key = now;
    };
    for (int first = 0; first < total; first += 32 * kSteps) {  // kSteps vectors of a lane on their way together
      uint4 q[kSteps];
      int at[kSteps];
#pragma unroll
      for (int u = 0; u < kSteps; ++u) {
        const int t = first + 32 * u + lane;
        at[u] = end;
        if (first + 32 * u >= total) continue;
        if (t < total) {
          const int group = best.groups[t >> each_bits];
          at[u] = warp_begin + ((group / 32 << each_bits) + (t & ((1 << each_bits) - 1))) * kStride + group % 32;
        }
        if (whole(at[u])) q[u] = __ldg(reinterpret_cast<const uint4*>(grid.row + grid.place(at[u])));
      }
#pragma unroll
      for (int u = 0; u < kSteps; ++u) {
        if (first + 32 * u >= total) break;
        uint32_t of[4] = {0, 0, 0, 0};
        if (at[u] < end) {
          if (!whole(at[u])) q[u] = edge_vector(grid.row, allowed, p.v, grid.place(at[u]));
          words(q[u], of);
          if (allowed && whole(at[u])) cut_out<T>(of, bytes_at<kValues>(allowed, grid.place(at[u]), p.v));
        }
        look_at(at[u], of);
      }
    }
    best.keep(p.top);
  }
  if constexpr (kWarps == 1) {
    const Normalizer normalizer(sums);
    if (lane == 0) write_scores(p, row, sums, normalizer, chosen);
    if (lane < p.top) write_top(p, row, lane, best.kept[lane], normalizer);
    return;
  }

  // The warps' sums and alternatives, these by their ranks among all: lists of `top` side by side, zeros where a part has
  // fewer logits. The first warp's ring and the second's have room for them.
  uint64_t* const lists = reinterpret_cast<uint64_t*>(rings);
  const auto rank_all = [&](int count, auto&& found) {
    __syncthreads();
    for (int i = threadIdx.x; i < count; i += kStride) {
      const uint64_t key = lists[i];
      int above = 0;
#pragma unroll 8
      for (int k = 0; k < count; ++k) above += lists[k] > key;
      if (key != 0 && above < p.top) found(above, key);
    }
  };
  static_assert(kWarps == 1 || (kWarps * kMostTop * 8 <= 2 * G::kRing * 16 && 8 * kMostTop * 8 <= G::kRing * 16), "lists fit");
  if (lane == 0) of_warps[warp] = sums;
  if (threadIdx.x < kMostTop) top_of_block[threadIdx.x] = 0;
  __syncthreads();  // the rings are free
  sums = of_team<kWarps>(of_warps[lane % kWarps]);
  const Normalizer normalizer(sums);
  if (blocks == 1 && threadIdx.x == 0) write_scores(p, row, sums, normalizer, chosen);
  if (p.top > 0) {
    if (lane < p.top) lists[warp * p.top + lane] = lane < best.count ? best.kept[lane] : 0;
    rank_all(kWarps * p.top, [&](int r, uint64_t key) {
      if (blocks == 1)
        write_top(p, row, r, key, normalizer);
      else
        top_of_block[r] = key;
    });
  }
  if (blocks == 1) return;

  // The cluster's first block does the same with the blocks'.
  if (threadIdx.x == 0) of_block = sums;
  cluster.sync();
  if (rank == 0) {
    sums = of_team<8>(lane % 8 < blocks ? *cluster.map_shared_rank(&of_block, lane % 8) : Sums{-infinity(), 0.0f, 0.0f});
    const Normalizer normalizer(sums);
    if (threadIdx.x == 0) write_scores(p, row, sums, normalizer, chosen);
    if (p.top > 0) {
      for (int i = threadIdx.x; i < 8 * kMostTop; i += kStride)
        if (i / kMostTop < blocks && i % kMostTop < p.top)
          lists[i / kMostTop * p.top + i % kMostTop] = cluster.map_shared_rank(top_of_block, i / kMostTop)[i % kMostTop];
      rank_all(blocks * p.top, [&](int r, uint64_t key) { write_top(p, row, r, key, normalizer); });
    }
  }
  cluster.sync();  // no block ends while its shared memory is read
}

// ---- the gradient ---------------------------------------------------------------------------------------

struct ScoresGrad {
  int64_t m, v;
  const float *grad_log_prob, *grad_entropy;  // null: zero
  const void* logits;
  int64_t stride;
  const void* actions;
  int action_dtype;
  const float *normalizer, *entropy;
  const uint8_t* allowed;
  int64_t allowed_stride;
  void* grad;
  const float* remainder;  // null: zero
};

// What a row's gradients have in common. With y = (l - normalizer) log2 e and the normalizer's remainder r, p = e^-r 2^y and the
// gradient of what was not chosen is - 2^y e^-r (g + h (entropy - r) + h ln 2 y): two values an instruction but for the power.
struct RowGrad {
  int action;  // negative: none whose gradient differs
  float g;
  uint64_t minus_base, a, b;
  RLENV_D RowGrad() {}
  RLENV_D RowGrad(const ScoresGrad& p, int64_t row) {
    const int64_t of_row = action_of(p.actions, p.action_dtype, row);
    check_flag(of_row >= p.v, kCheckActionRange);
    action = of_row < 0 ? -1 : int(of_row < p.v ? of_row : p.v);
    const float normalizer = __ldg(p.normalizer + row), entropy = __ldg(p.entropy + row);
    const float h = p.grad_entropy ? __ldg(p.grad_entropy + row) : 0.0f;
    g = p.grad_log_prob && action >= 0 ? __ldg(p.grad_log_prob + row) : 0.0f;
    if (action >= p.v) g = not_a_number();
    float rest = 0.0f, scale = 1.0f;
    if (p.remainder) rest = __ldg(p.remainder + row), scale = expf(-rest);
    const bool none = normalizer == -infinity();
    if (none) action = -1;
    const float base = none ? 0.0f : normalizer, of_p = none ? 0.0f : -scale * (g + h * (entropy - rest)),
                of_y = none ? 0.0f : -scale * h * kLn2;
    minus_base = pair_of(-base, -base), a = pair_of(of_p, of_p), b = pair_of(of_y, of_y);
  }
  RLENV_D float2 without_choice(uint64_t l) const {
    const uint64_t y = powers_of(l, minus_base);
    const float2 of = values_of(y);
    return values_of(multiply_pairs(pair_of(exp2_fast(of.x), exp2_fast(of.y)), multiply_add_pairs(b, y, a)));
  }
  RLENV_D float of_choice(float l) const { return l == -infinity() ? 0.0f : g; }
  // Another lane's, among kLanes neighbouring ones.
  template <int kLanes>
  RLENV_D RowGrad of_lane(int lane) const {
    RowGrad r;
    const float base = __shfl_sync(0xffffffffu, values_of(minus_base).x, lane, kLanes),
                of_p = __shfl_sync(0xffffffffu, values_of(a).x, lane, kLanes), of_y = __shfl_sync(0xffffffffu, values_of(b).x, lane, kLanes);
    r.action = __shfl_sync(0xffffffffu, action, lane, kLanes), r.g = __shfl_sync(0xffffffffu, g, lane, kLanes);
    r.minus_base = pair_of(base, base), r.a = pair_of(of_p, of_p), r.b = pair_of(of_y, of_y);
    return r;
  }
};

RLENV_D void store_value(float* to, float x) { *to = x; }
RLENV_D void store_value(__nv_bfloat16* to, float x) { *to = __float2bfloat16_rn(x); }

// Rows of few actions: kLanes neighbouring lanes a row, as in the forward pass.
template <typename T, int kLanes, int kEach>
__global__ void __launch_bounds__(256) few_scores_grad_kernel(const __grid_constant__ ScoresGrad p, int turns) {
  constexpr int kAtOnce = 32 / kLanes;
  const int sub = threadIdx.x % kLanes, team = threadIdx.x % 32 / kLanes, m = int(p.m);
  const int first = int(blockIdx.x * 8 + threadIdx.x / 32) * (kAtOnce * turns), own = first + sub * kAtOnce + team;
  RowGrad of_own;
  if (sub < turns && own < m) of_own = RowGrad(p, own);
#pragma unroll 1
  for (int turn = 0; turn < turns && first + turn * kAtOnce < m; ++turn) {
    const int at = first + turn * kAtOnce + team, row = min(at, m - 1);
    float x[kEach];
    few_logits<kLanes, kEach, T>(p, row, sub, x);
    const RowGrad of = of_own.of_lane<kLanes>(turn);
    T* const grad = static_cast<T*>(p.grad) + row * p.v + sub;
    const int left = at < m ? int(p.v) - sub : 0, chosen = of.action - sub;
#pragma unroll
    for (int i = 0; i < kEach; i += 2) {
      float2 g = of.without_choice(pair_of(x[i], x[i + 1]));
      if (chosen == kLanes * i) g.x += of.of_choice(x[i]);
      if (chosen == kLanes * (i + 1)) g.y += of.of_choice(x[i + 1]);
      if (kLanes * i < left) store_value(grad + kLanes * i, g.x);
      if (kLanes * (i + 1) < left) store_value(grad + kLanes * (i + 1), g.y);
    }
  }
}

// A warp a run of a row of the gradient, kVectors a lane on 16-byte boundaries. kAlike: the logits' rows lie on the
// boundaries as the gradient's do. What counts is bytes on their way: 4 vectors with 40 warps an SM (4,096 x 16,384 bf16 48
// us; 2 vectors with 56 warps 51), with masks, whose bytes take registers too, 2 with 48 (4,096 x 32,771 120 us; 4 with 40
// warps 139, 2 with 56 warps 143), and rows between the boundaries 2 with 56 (60 us; 4 with 40 warps 68).
template <bool kAlike, bool kMasked>
struct Run {
  static constexpr int kVectors = kAlike && !kMasked ? 4 : 2, kBlocks = kMasked ? 6 : kAlike ? 5 : 7;  // of 8 warps, an SM's
};
template <typename T, bool kAlike, bool kMasked>
__global__ void __launch_bounds__(256, Run<kAlike, kMasked>::kBlocks)
scores_grad_kernel(const __grid_constant__ ScoresGrad p, uint32_t runs) {
  constexpr int kValues = Grid<T>::kValues, kVectors = Run<kAlike, kMasked>::kVectors, kRun = 32 * kVectors;
  const uint32_t warp = blockIdx.x * 8 + threadIdx.x / 32, of_row = warp / runs;
  const int64_t row = of_row;
  if (row >= p.m) return;
  const int lane = threadIdx.x % 32, first = int(warp - of_row * runs) * kRun + lane;
  const T* const logits = static_cast<const T*>(p.logits) + row * p.stride;
  const uint8_t* const allowed = p.allowed ? p.allowed + row * p.allowed_stride : nullptr;
  T* const grad = static_cast<T*>(p.grad) + row * p.v;
  const Grid<T> to(grad, p.v);
  const int vectors = int(to.vectors());
  const int first_whole = to.skip > 0, last_whole = (to.skip + p.v) % kValues ? vectors - 1 : vectors;
  uint32_t w[kVectors][4];
  uint2 bytes[kVectors];
#pragma unroll
  for (int r = 0; r < kVectors; ++r) {
    const int i = first + 32 * r;
    const int64_t j0 = to.place(i);
    const bool inside = i >= first_whole && i < last_whole && (kAlike || (j0 > 0 && j0 + kValues < p.v));
    if (inside) {
      const uint4 q = kAlike ? __ldg(reinterpret_cast<const uint4*>(logits + j0)) : words_between(logits, j0);
      w[r][0] = q.x, w[r][1] = q.y, w[r][2] = q.z, w[r][3] = q.w;
      if (kMasked) bytes[r] = bytes_at<kValues>(allowed, j0, p.v);
    }
  }
  const RowGrad of(p, row);
#pragma unroll
  for (int r = 0; r < kVectors; ++r) {
    const int i = first + 32 * r;
    if (i >= vectors) break;
    const int64_t j0 = to.place(i);
    const bool whole = i >= first_whole && i < last_whole;
    if (whole && (kAlike || (j0 > 0 && j0 + kValues < p.v))) {
      if (kMasked) cut_out<T>(w[r], bytes[r]);
    } else {
      const uint4 q = edge_vector(logits, allowed, p.v, j0);
      w[r][0] = q.x, w[r][1] = q.y, w[r][2] = q.z, w[r][3] = q.w;
    }
    float x[kValues];
#pragma unroll
    for (int k = 0; k < kValues / 2; ++k) {
      const float2 v = of.without_choice(word_pair<T>(w[r], k));
      x[2 * k] = v.x, x[2 * k + 1] = v.y;
    }
    const int64_t chosen = of.action - j0;
    if (chosen >= 0 && chosen < kValues) {
#pragma unroll
      for (int j = 0; j < kValues; ++j)
        if (j == chosen) x[j] += of.of_choice(word_value<T>(w[r], j));
    }
    if (whole) {
      if constexpr (sizeof(T) == 4) {
        *reinterpret_cast<float4*>(grad + j0) = make_float4(x[0], x[1], x[2], x[3]);
      } else {
        uint32_t out[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const __nv_bfloat162 pair = __floats2bfloat162_rn(x[2 * k], x[2 * k + 1]);
          out[k] = *reinterpret_cast<const uint32_t*>(&pair);
        }
        *reinterpret_cast<uint4*>(grad + j0) = make_uint4(out[0], out[1], out[2], out[3]);
      }
    } else {
#pragma unroll
      for (int j = 0; j < kValues; ++j)
        if (j0 + j >= 0 && j0 + j < p.v) store_value(grad + j0 + j, x[j]);
    }
  }
}

// ---- host -----------------------------------------------------------------------------------------------

bool at_multiple(const void* p, int size) { return reinterpret_cast<uintptr_t>(p) % size == 0; }

template <typename T, int kLanes, int kEach>
int few_scores(const Scores& p, cudaStream_t s) {
  few_scores_kernel<T, kLanes, kEach><<<unsigned((p.m * kLanes + 255) / 256), 256, 0, s>>>(p);
  return launch_status();
}
template <typename T>
int few_scores_of(const Scores& p, cudaStream_t s) {
  if (p.v <= 8) return few_scores<T, 1, 8>(p, s);
  if (p.v <= 16) return few_scores<T, 2, 8>(p, s);
  if (p.v <= 32) return few_scores<T, 4, 8>(p, s);
  // Rows that are many by few lanes (169,089 of 100 float32 18 us, by 16 lanes 24), so that a row's end is cheap; others by a warp,
  // whose lanes have less to do one after the other (2,000 of 100 with four alternatives 3.0 us, by 8 lanes 4.8).
  const bool many = p.m > 8192;
  if (p.v <= 64) return many ? few_scores<T, 4, 16>(p, s) : few_scores<T, 32, 2>(p, s);
  if (p.v <= 128) return many ? few_scores<T, 8, 16>(p, s) : few_scores<T, 32, 4>(p, s);
  // Alternatives by a warp (169,089 of 200 float32 with eight 98 us, by 16 lanes 206; without any 43 and 32).
  if (p.v <= 256) return p.top == 0 ? few_scores<T, 16, 16>(p, s) : few_scores<T, 32, 8>(p, s);
  if (p.v <= 512) return few_scores<T, 32, 16>(p, s);
  return few_scores<T, 32, 32>(p, s);
}

// A warp takes rows in turns, as many as leave 80 warps to an SM, twice what it holds (198,564 of 200 bf16 42 us, all rows in
// turns of their own 70).
template <typename T, int kLanes, int kEach>
int few_scores_grad(const ScoresGrad& p, cudaStream_t s) {
  constexpr int kAtOnce = 32 / kLanes;
  const int64_t most = p.m / (kAtOnce * 148 * 80);
  const int turns = most < 1 ? 1 : most > kLanes ? kLanes : int(most), rows = kAtOnce * 8 * turns;
  few_scores_grad_kernel<T, kLanes, kEach><<<unsigned((p.m + rows - 1) / rows), 256, 0, s>>>(p, turns);
  return launch_status();
}
template <typename T>
int few_scores_grad_of(const ScoresGrad& p, cudaStream_t s) {
  if (p.v <= 8) return few_scores_grad<T, 1, 8>(p, s);
  if (p.v <= 16) return few_scores_grad<T, 2, 8>(p, s);
  if (p.v <= 32) return few_scores_grad<T, 4, 8>(p, s);
  if (p.v <= 64) return few_scores_grad<T, 8, 8>(p, s);
  if (p.v <= 128) return few_scores_grad<T, 16, 8>(p, s);  // 198,564 of 106 bf16 24 us, by 8 lanes 28
  if (p.v <= 256) return few_scores_grad<T, 16, 16>(p, s);  // of 200 42 us, by 32 lanes 46
  if (p.v <= 512) return few_scores_grad<T, 32, 16>(p, s);
  return few_scores_grad<T, 32, 32>(p, s);
}

template <typename T, int kWarps>
int scores(const Scores& p, int blocks, cudaStream_t s) {
  using G = Team<kWarps>;
  cudaLaunchConfig_t config{};
  config.gridDim = dim3(unsigned((p.m + G::kRows - 1) / G::kRows * blocks));
  config.blockDim = dim3(G::kThreads);
  config.dynamicSmemBytes = G::kShared;
  config.stream = s;
  cudaLaunchAttribute cluster{};
  cluster.id = cudaLaunchAttributeClusterDimension;
  cluster.val.clusterDim.x = unsigned(blocks), cluster.val.clusterDim.y = cluster.val.clusterDim.z = 1;
  config.attrs = &cluster, config.numAttrs = blocks > 1 ? 1 : 0;
  if (G::kShared > 32 * 1024)
    if (cudaError_t e = cudaFuncSetAttribute(scores_kernel<T, kWarps>, cudaFuncAttributeMaxDynamicSharedMemorySize, G::kShared))
      return int(e);
  const cudaError_t e = cudaLaunchKernelEx(&config, scores_kernel<T, kWarps>, p);
  return e == cudaSuccess ? launch_status() : int(e);
}

template <typename T>
int scores_of(const Scores& p, cudaStream_t s) {
  constexpr int kValues = Grid<T>::kValues;
  if (p.v <= 1024) return few_scores_of<T>(p, s);
  // Warps a row. One for short rows that are many: what a row's end costs, its warps' joining above all, is paid by more rows at a
  // time (5,000 of 5,000 bf16 with eight alternatives 24 us, by four warps 37; 9,000 of 15,000 54 and 58; 1,000 of 3,000 7.9 and
  // 9.8). Four for long ones, whose warps then end at different times (4,096 of 32,768 bf16 49 us, by one warp 56; 2,400 of 60,000
  // 53 and 68; 1,300 of 100,000 53 and 91), and of fewer rows (567 of 4,341 float32 7.9, by 16 warps 18.0; 300 of 10,000 8.4
  // and 15.6). Sixteen, and a cluster of blocks that have a turn each, of few long rows (one row of 50,021 bf16 5.0 us, one block
  // 6.7; 20 of 30,000 float32 8.2, with a vector a thread 11.0).
  const int64_t vectors = p.v / kValues;
  if ((vectors <= 512 && p.m >= 4 * 148) || (vectors <= 2048 && p.m >= 16 * 148)) return scores<T, 1>(p, 1, s);
  if (p.m >= 2 * 148 || vectors <= 256) return scores<T, 4>(p, 1, s);
  int blocks = 1;
  while (blocks < 8 && p.m * 16 * blocks < 8 * 148 && vectors > 2048 * blocks) blocks *= 2;
  return scores<T, 16>(p, blocks, s);
}

template <typename T>
int scores_grad_of(const ScoresGrad& p, cudaStream_t s) {
  constexpr int kValues = Grid<T>::kValues;
  const int64_t vectors = (p.v + 2 * kValues - 2) / kValues;
  const bool alike = p.stride % kValues == p.v % kValues && reinterpret_cast<uintptr_t>(p.logits) % 16 ==
                     reinterpret_cast<uintptr_t>(p.grad) % 16;
  // Where logits and gradient lie differently on the boundaries, rows of lanes' single values are quicker for longer (52,413 of
  // 1,000 bf16 54 us, by vectors 73, and 42 where they lie alike; 100,000 of 300 alike 40 and 70, of 512 47 and 54).
  if (p.v <= (alike ? 512 : 1024)) return few_scores_grad_of<T>(p, s);
  const auto run = [&](auto is_alike, auto is_masked) {
    constexpr bool kAlike = decltype(is_alike)::value, kMasked = decltype(is_masked)::value;
    constexpr int kRun = 32 * Run<kAlike, kMasked>::kVectors;
    const int64_t runs = (vectors + kRun - 1) / kRun;
    scores_grad_kernel<T, kAlike, kMasked><<<unsigned((p.m * runs + 7) / 8), 256, 0, s>>>(p, uint32_t(runs));
  };
  if (alike && p.allowed)
    run(std::true_type(), std::true_type());
  else if (alike)
    run(std::true_type(), std::false_type());
  else if (p.allowed)
    run(std::false_type(), std::true_type());
  else
    run(std::false_type(), std::false_type());
  return launch_status();
}

bool scores_sizes(int dtype, int64_t m, int64_t v, int64_t stride, int action_dtype, int64_t allowed_stride) {
  return (dtype == RLENV_F32 || dtype == RLENV_BF16) && m >= 0 && v >= 1 && v <= (int64_t(1) << 31) - 64 &&
         m < (int64_t(1) << 26) && m * v < (int64_t(1) << 40) && stride >= 0 && allowed_stride >= 0 &&
         valid_dtype(action_dtype);
}
int action_size(int dtype) { return dtype == RLENV_I64 ? 8 : dtype == RLENV_I32 ? 4 : 1; }

}  // namespace
}  // namespace rlenv

extern "C" {

int rlenv_log_probs_forward(int dtype, int64_t m, int64_t v, const void* logits, int64_t stride, const void* actions,
                            int action_dtype, const uint8_t* allowed, int64_t allowed_stride, float* log_prob,
                            float* entropy, float* normalizer, int top, int64_t* top_actions, float* top_log_probs,
                            void* stream) {
  return rlenv_log_probs_forward_remainder(dtype, m, v, logits, stride, actions, action_dtype, allowed, allowed_stride, log_prob,
                                           entropy, normalizer, nullptr, top, top_actions, top_log_probs, stream);
}

int rlenv_log_probs_forward_remainder(int dtype, int64_t m, int64_t v, const void* logits, int64_t stride, const void* actions,
                                      int action_dtype, const uint8_t* allowed, int64_t allowed_stride, float* log_prob,
                                      float* entropy, float* normalizer, float* remainder, int top, int64_t* top_actions,
                                      float* top_log_probs, void* stream) {
  using namespace rlenv;
  if (!scores_sizes(dtype, m, v, stride, action_dtype, allowed_stride) || top < 0 || top > kMostTop || top > v)
    return RLENV_EINVAL;
  if (m == 0) return RLENV_OK;
  if (!logits || !actions || !log_prob || !entropy || !normalizer || (top > 0 && (!top_actions || !top_log_probs)))
    return RLENV_EINVAL;
  if (!at_multiple(logits, dtype == RLENV_F32 ? 4 : 2) || !at_multiple(actions, action_size(action_dtype)) ||
      !at_multiple(log_prob, 4) || !at_multiple(entropy, 4) || !at_multiple(normalizer, 4) || !at_multiple(remainder, 4) ||
      !at_multiple(top_actions, 8) || !at_multiple(top_log_probs, 4))
    return RLENV_EINVAL;
  const Scores p{m, v, logits, stride, actions, action_dtype, allowed, allowed_stride, log_prob, entropy, normalizer,
                 top, top_actions, top_log_probs, remainder};
  return dtype == RLENV_F32 ? scores_of<float>(p, as_stream(stream)) : scores_of<__nv_bfloat16>(p, as_stream(stream));
}

int rlenv_log_probs_backward(int dtype, int64_t m, int64_t v, const float* grad_log_prob, const float* grad_entropy,
                             const void* logits, int64_t stride, const void* actions, int action_dtype,
                             const float* normalizer, const float* entropy, const uint8_t* allowed, int64_t allowed_stride,
                             void* grad, void* stream) {
  return rlenv_log_probs_backward_remainder(dtype, m, v, grad_log_prob, grad_entropy, logits, stride, actions, action_dtype,
                                            normalizer, nullptr, entropy, allowed, allowed_stride, grad, stream);
}

int rlenv_log_probs_backward_remainder(int dtype, int64_t m, int64_t v, const float* grad_log_prob, const float* grad_entropy,
                                       const void* logits, int64_t stride, const void* actions, int action_dtype,
                                       const float* normalizer, const float* remainder, const float* entropy,
                                       const uint8_t* allowed, int64_t allowed_stride, void* grad, void* stream) {
  using namespace rlenv;
  if (!scores_sizes(dtype, m, v, stride, action_dtype, allowed_stride)) return RLENV_EINVAL;
  if (m == 0) return RLENV_OK;
  const int size = dtype == RLENV_F32 ? 4 : 2;
  if (!logits || !actions || !normalizer || !entropy || !grad || !at_multiple(logits, size) || !at_multiple(grad, size) ||
      !at_multiple(actions, action_size(action_dtype)) || !at_multiple(normalizer, 4) || !at_multiple(entropy, 4) ||
      !at_multiple(grad_log_prob, 4) || !at_multiple(grad_entropy, 4) || !at_multiple(remainder, 4))
    return RLENV_EINVAL;
  const ScoresGrad p{m, v, grad_log_prob, grad_entropy, logits, stride, actions, action_dtype, normalizer, entropy, allowed,
                     allowed_stride, grad, remainder};
  return dtype == RLENV_F32 ? scores_grad_of<float>(p, as_stream(stream))
                            : scores_grad_of<__nv_bfloat16>(p, as_stream(stream));
}

}  // extern "C"
