// Scores of actions: the log-probability of a chosen one, the entropy and the best alternatives of rows of logits, and
// their gradient. With the largest logit b of a row (of those allowed; others count as -infinity),
//     S = sum e^(l - b),   W = sum e^(l - b) (l - b),   normalizer = b + log S,   entropy = log S - W / S,
// and sums over parts of a row join: (b, S, W) moves to a larger b' by d = b - b': (e^d S, e^d (W + S d)).
// The gradient: g ([j = action] - p_j) - h p_j (log p_j + entropy), p_j = e^(l_j - normalizer).
//
// Bound by memory: a row is read once, held in registers between its largest value, its sums and its alternatives.
#include <cooperative_groups.h>
#include <cuda_bf16.h>

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

// Two float32 values side by side: sm_100 adds and multiplies them in one instruction.
RLENV_D uint64_t pair_of(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
RLENV_D float2 values_of(uint64_t p) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(p));
  return r;
}
RLENV_D uint64_t add_pairs(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
RLENV_D uint64_t multiply_pairs(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
RLENV_D uint64_t multiply_add_pairs(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
RLENV_D float exp2_fast(float x) {  // within 2 ulp, 0 where float32's normal numbers end
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
constexpr float kLog2E = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

// Logits are ordered by value, ties by the lower place: as one whole number, larger first. 0 stands below all, NaN
// above.
RLENV_D uint32_t order_of(float x) {
  if (x != x) return 0xffffffffu;
  const uint32_t b = x == 0.0f ? 0u : __float_as_uint(x);  // both zeros are one
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
RLENV_D float value_of(uint32_t order) {
  return __uint_as_float(order & 0x80000000u ? order & 0x7fffffffu : ~order);
}
RLENV_D uint64_t key_of(float x, uint32_t place) { return uint64_t(order_of(x)) << 32 | ~place; }

// l - normalizer, also where both are -infinity.
RLENV_D float log_prob_of(float l, float normalizer) {
  return l == -infinity() && normalizer == -infinity() ? l : l - normalizer;
}

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
RLENV_D void add(Sums& a, float l, float base) {
  const float d = larger(l - base, kFar), e = __expf(d);
  a.s += e;
  a.w = fmaf(e, d, a.w);
}

RLENV_D float normalizer_of(const Sums& a) { return base_of(a.m) + logf(a.s); }

template <typename T>
RLENV_D void write_scores(const Scores& p, int64_t row, const Sums& sums) {
  const float normalizer = normalizer_of(sums);
  p.normalizer[row] = normalizer;
  p.entropy[row] = sums.s == 0.0f ? 0.0f : logf(sums.s) - sums.w / sums.s;
  const int64_t a = action_of(p.actions, p.action_dtype, row);
  check_flag(a >= p.v, kCheckActionRange);
  float lp = 0.0f;
  if (a >= p.v) {
    lp = not_a_number();
  } else if (a >= 0) {
    const bool open = !p.allowed || p.allowed[row * p.allowed_stride + a];
    lp = log_prob_of(open ? value_at(static_cast<const T*>(p.logits) + row * p.stride + a) : -infinity(), normalizer);
  }
  p.log_prob[row] = lp;
}
RLENV_D void write_top(const Scores& p, int64_t row, int rank, uint64_t key, float normalizer) {
  p.top_actions[row * p.top + rank] = int64_t(uint32_t(~uint32_t(key)));
  p.top_log_probs[row * p.top + rank] = log_prob_of(value_of(uint32_t(key >> 32)), normalizer);
}

// ---- few actions: a row is the work of kLanes neighbouring lanes -----------------------------------------

constexpr int kEach = 8;  // logits of a lane
template <typename T, int kLanes>
__global__ void __launch_bounds__(256) few_scores_kernel(const __grid_constant__ Scores p) {
  const int sub = threadIdx.x % kLanes;
  const int64_t at = (int64_t(blockIdx.x) * 256 + threadIdx.x) / kLanes, row = at < p.m ? at : p.m - 1;
  const T* const logits = static_cast<const T*>(p.logits) + row * p.stride;
  const uint8_t* const allowed = p.allowed ? p.allowed + row * p.allowed_stride : nullptr;
  const int v = int(p.v);
  float x[kEach];
  Sums sums{-infinity(), 0.0f, 0.0f};
#pragma unroll
  for (int i = 0; i < kEach; ++i) {
    const int j = sub + kLanes * i;
    x[i] = j < v && (!allowed || allowed[j]) ? value_at(logits + j) : -infinity();
  }
#pragma unroll
  for (int i = 0; i < kEach; ++i) sums.m = larger(sums.m, x[i]);
#pragma unroll
  for (int d = kLanes / 2; d > 0; d /= 2) sums.m = larger(sums.m, __shfl_xor_sync(0xffffffffu, sums.m, d));
#pragma unroll
  for (int i = 0; i < kEach; ++i) add(sums, x[i], base_of(sums.m));
#pragma unroll
  for (int d = kLanes / 2; d > 0; d /= 2) {
    sums.s += __shfl_xor_sync(0xffffffffu, sums.s, d);
    sums.w += __shfl_xor_sync(0xffffffffu, sums.w, d);
  }
  if (sub == 0 && at < p.m) write_scores<T>(p, row, sums);
  if (p.top == 0) return;
  const float normalizer = normalizer_of(sums);
  uint32_t taken = 0;
  for (int r = 0; r < p.top; ++r) {
    uint64_t best = 0;
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
      const int j = sub + kLanes * i;
      const uint64_t key = j < v && !(taken >> i & 1) ? key_of(x[i], j) : 0;
      best = key > best ? key : best;
    }
#pragma unroll
    for (int d = kLanes / 2; d > 0; d /= 2) {
      const uint64_t other = __shfl_xor_sync(0xffffffffu, best, d);
      best = other > best ? other : best;
    }
    const int j = int(~uint32_t(best));
    if (j % kLanes == sub) taken |= 1u << (j / kLanes);
    if (sub == 0 && at < p.m) write_top(p, row, r, best, normalizer);
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
template <typename T>
RLENV_D uint32_t word_of(float x) {  // x in each place
  if constexpr (sizeof(T) == 4) return __float_as_uint(x);
  const __nv_bfloat162 p = __float2bfloat162_rn(x);
  return *reinterpret_cast<const uint32_t*>(&p);
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
RLENV_D bool any_reaches(uint32_t w, uint32_t least) {  // a place that is not below least's
  if constexpr (sizeof(T) == 4) return !(__uint_as_float(w) < __uint_as_float(least));
  return __hgeu2_mask(as_bf162(w), as_bf162(least)) != 0;
}
// log2 e^(l - base) of two logits. What lies further below than kFar counts as that: it adds nothing, and -infinity times
// nothing would be NaN.
RLENV_D uint64_t powers_of(uint64_t l, uint64_t minus_base) {
  const float2 d = values_of(add_pairs(l, minus_base));
  return multiply_pairs(pair_of(larger(d.x, kFar), larger(d.y, kFar)), pair_of(kLog2E, kLog2E));
}
template <typename T>
RLENV_D constexpr uint32_t empty_word() {  // -infinity
  return sizeof(T) == 4 ? 0xff800000u : 0xff80ff80u;
}

// The kValues bytes of `allowed` from place j0 on, all of them in the row, as two words.
template <int kValues>
RLENV_D uint2 bytes_at(const uint8_t* allowed, int64_t j0, int64_t v) {
  const uint8_t* const at = allowed + j0;
  const unsigned off = unsigned(reinterpret_cast<uintptr_t>(at) % 4);
  uint2 b = make_uint2(0, 0);
  if (off == 0) {
    const uint32_t* const words = reinterpret_cast<const uint32_t*>(at);
    b.x = __ldg(words);
    if (kValues == 8) b.y = __ldg(words + 1);
  } else if (j0 >= 4 && j0 + kValues + 4 <= v) {  // the words around them are in the row too
    const uint32_t* const words = reinterpret_cast<const uint32_t*>(at - off);
    const uint32_t w0 = __ldg(words), w1 = __ldg(words + 1);
    b.x = __funnelshift_r(w0, w1, 8 * off);
    if (kValues == 8) b.y = __funnelshift_r(w1, __ldg(words + 2), 8 * off);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      b.x |= uint32_t(at[i]) << 8 * i;
      if (kValues == 8) b.y |= uint32_t(at[4 + i]) << 8 * i;
    }
  }
  return b;
}

// Vector i of a row in 32-bit words, -infinity where a place is not allowed or not in the row.
template <typename T>
RLENV_D void load_vector(const Grid<T>& grid, const uint8_t* allowed, int64_t i, uint32_t (&w)[4]) {
  constexpr int kValues = Grid<T>::kValues;
  const int64_t j0 = grid.place(i);
  if (j0 >= 0 && j0 + kValues <= grid.v) {
    const uint4 q = __ldg(reinterpret_cast<const uint4*>(grid.row + j0));
    w[0] = q.x, w[1] = q.y, w[2] = q.z, w[3] = q.w;
    if (allowed) {
      const uint2 b = bytes_at<kValues>(allowed, j0, grid.v);
      const uint32_t none[2] = {__vcmpeq4(b.x, 0), __vcmpeq4(b.y, 0)};  // 0xff for what is not allowed
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const uint32_t mask = kValues == 8 ? __byte_perm(none[k / 2], 0, k % 2 ? 0x3322 : 0x1100)
                                           : __byte_perm(none[0], 0, 0x1111 * k);
        w[k] = (w[k] & ~mask) | (empty_word<T>() & mask);
      }
    }
  } else {
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      w[k] = 0;
#pragma unroll
      for (int h = 0; h < kValues / 4; ++h) {
        const int64_t j = j0 + k * (kValues / 4) + h;
        const bool open = j >= 0 && j < grid.v && (!allowed || allowed[j]);
        const float x = open ? value_at(grid.row + j) : -infinity();
        w[k] |= sizeof(T) == 4 ? __float_as_uint(x) : __float_as_uint(x) >> 16 << 16 * h;
      }
    }
  }
}

// A team of kThreads threads, a warp or a block, in 32 groups of neighbours.
template <int kThreads>
struct Team {
  static constexpr int kWarps = kThreads / 32, kBlock = kThreads == 32 ? 256 : kThreads, kRows = kBlock / kThreads;
  static constexpr int kRoom = kThreads == 32 ? 128 : 4 * kThreads;  // alternatives looked at
  struct Shared {
    float groups[32], sums[2 * kWarps];
    uint64_t keys[kRoom], top[kMostTop];
    uint32_t count;
    float of_block[3];
  };
  static RLENV_D void sync() {
    if constexpr (kWarps == 1)
      __syncwarp();
    else
      __syncthreads();
  }
  // The team's largest key; room holds kWarps of them.
  static RLENV_D uint64_t most(uint64_t x, uint64_t* room) {
#pragma unroll
    for (int d = 16; d > 0; d /= 2) {
      const uint64_t y = __shfl_xor_sync(0xffffffffu, x, d);
      x = y > x ? y : x;
    }
    if constexpr (kWarps > 1) {
      if (threadIdx.x % 32 == 0) room[threadIdx.x / 32] = x;
      __syncthreads();
      x = room[threadIdx.x % kWarps];
#pragma unroll
      for (int d = kWarps / 2; d > 0; d /= 2) {
        const uint64_t y = __shfl_xor_sync(0xffffffffu, x, d);
        x = y > x ? y : x;
      }
      __syncthreads();
    }
    return x;
  }
};

// The n-th largest of a warp's values, known to all lanes: sorted by exchanges with lanes at growing distances
// (Batcher 1968).
RLENV_D float nth_largest(float x, int n) {
  const int lane = threadIdx.x % 32;
  uint32_t v = order_of(x);
#pragma unroll
  for (int size = 2; size <= 32; size *= 2)
#pragma unroll
    for (int d = size / 2; d > 0; d /= 2) {
      const uint32_t other = __shfl_xor_sync(0xffffffffu, v, d);
      v = ((lane & d) == 0) == ((lane & size) == 0) ? max(v, other) : min(v, other);
    }
  return value_of(__shfl_sync(0xffffffffu, v, n - 1));
}

// kThreads threads with room for kVectors vectors each; longer parts of a row go tile by tile, and are read again for
// their sums. A cluster's blocks have a part of the row each.
//
// The alternatives: the n-th largest of the 32 groups' largest logits has n logits at least that are not below it, and as
// a rule few more. These are collected and their ranks counted; where they are too many (a row of equal logits, or all
// large ones in one group) they are found one after the other.
template <typename T, int kThreads, int kVectors>
__global__ void __launch_bounds__(Team<kThreads>::kBlock) scores_kernel(const __grid_constant__ Scores p) {
  using G = Team<kThreads>;
  constexpr int kValues = Grid<T>::kValues, kTile = kThreads * kVectors;
  __shared__ typename G::Shared shared[G::kRows];
  auto& sh = shared[threadIdx.x / kThreads];
  cg::cluster_group cluster = cg::this_cluster();
  const int blocks = kThreads == 32 ? 1 : int(cluster.num_blocks()), rank = blocks > 1 ? int(cluster.block_rank()) : 0;
  const int at = threadIdx.x % kThreads, lane = threadIdx.x % 32;
  const int64_t row = kThreads == 32 ? int64_t(blockIdx.x) * G::kRows + threadIdx.x / 32 : blockIdx.x / blocks;
  if (row >= p.m) return;  // a warp
  const Grid<T> grid(static_cast<const T*>(p.logits) + row * p.stride, p.v);
  const uint8_t* const allowed = p.allowed ? p.allowed + row * p.allowed_stride : nullptr;
  const int vectors = int(grid.vectors()), part = (vectors + blocks - 1) / blocks, begin = min(rank * part, vectors),
            end = min(begin + part, vectors);
  const bool one_tile = end - begin <= kTile;

  uint32_t w[kVectors][4];
  const auto load_tile = [&](int from) {
#pragma unroll
    for (int r = 0; r < kVectors; ++r) {
      const int i = from + r * kThreads + at;
      if (i < end) {
        load_vector(grid, allowed, i, w[r]);
      } else {
#pragma unroll
        for (int k = 0; k < 4; ++k) w[r][k] = empty_word<T>();
      }
    }
  };
  // f(r) for the tile's vectors of this thread; the same ones are left out by all threads.
  const auto each_vector = [&](int from, auto&& f) {
#pragma unroll
    for (int r = 0; r < kVectors; ++r)
      if (from + r * kThreads < end) f(r);
  };
  uint32_t most = empty_word<T>();
  for (int from = begin; from < end; from += kTile) {
    load_tile(from);
    each_vector(from, [&](int r) {
      most = larger_words<T>(most, larger_words<T>(larger_words<T>(w[r][0], w[r][1]), larger_words<T>(w[r][2], w[r][3])));
    });
  }
  const float own_most = largest_of<T>(most);
  float group = own_most;
  if constexpr (kThreads > 32) {
#pragma unroll
    for (int d = (kThreads / 32) / 2; d > 0; d /= 2) group = larger(group, __shfl_xor_sync(0xffffffffu, group, d));
    if (at % (kThreads / 32) == 0) sh.groups[at / (kThreads / 32)] = group;
  }
  if (at == 0) sh.count = 0;
  G::sync();
  if constexpr (kThreads > 32) group = sh.groups[lane];
  Sums sums{group, 0.0f, 0.0f};
#pragma unroll
  for (int d = 16; d > 0; d /= 2) sums.m = larger(sums.m, __shfl_xor_sync(0xffffffffu, sums.m, d));
  const float base = base_of(sums.m);
  const float least = p.top > 0 ? nth_largest(group, p.top) : 0.0f;

  const uint32_t reach = word_of<T>(least);
  const uint64_t minus_base = pair_of(-base, -base);
  const bool mine = p.top > 0 && !(own_most < least);
  uint64_t s2 = 0, w2 = 0;
  for (int from = begin; from < end; from += kTile) {
    if (!one_tile) load_tile(from);
    if (mine)
      each_vector(from, [&](int r) {
#pragma unroll
        for (int k = 0; k < 4; ++k)
          if (any_reaches<T>(w[r][k], reach)) {
#pragma unroll
            for (int h = 0; h < kValues / 4; ++h) {
              const int j = k * (kValues / 4) + h;
              const float x = word_value<T>(w[r], j);
              const int64_t place = grid.place(from + r * kThreads + at) + j;
              if (x < least || place < 0 || place >= p.v || from + r * kThreads + at >= end) continue;
              const uint32_t slot = atomicAdd(&sh.count, 1u);
              if (slot < G::kRoom) sh.keys[slot] = key_of(x, uint32_t(place));
            }
          }
      });
    each_vector(from, [&](int r) {
#pragma unroll
      for (int i = 0; i < kValues / 2; ++i) {
        const uint64_t y = powers_of(word_pair<T>(w[r], i), minus_base);
        const float2 of = values_of(y);
        const uint64_t e = pair_of(exp2_fast(of.x), exp2_fast(of.y));
        s2 = add_pairs(s2, e), w2 = multiply_add_pairs(e, y, w2);
      }
    });
  }
  const float2 s_own = values_of(s2), w_own = values_of(w2);
  sums.s = s_own.x + s_own.y, sums.w = (w_own.x + w_own.y) * kLn2;
#pragma unroll
  for (int d = 16; d > 0; d /= 2) {
    sums.s += __shfl_xor_sync(0xffffffffu, sums.s, d);
    sums.w += __shfl_xor_sync(0xffffffffu, sums.w, d);
  }
  if (kThreads > 32 && lane == 0) sh.sums[at / 32] = sums.s, sh.sums[G::kWarps + at / 32] = sums.w;
  G::sync();
  if constexpr (kThreads > 32) {
    sums.s = sh.sums[lane % G::kWarps], sums.w = sh.sums[G::kWarps + lane % G::kWarps];
#pragma unroll
    for (int d = G::kWarps / 2; d > 0; d /= 2) {
      sums.s += __shfl_xor_sync(0xffffffffu, sums.s, d);
      sums.w += __shfl_xor_sync(0xffffffffu, sums.w, d);
    }
  }
  const bool alone = kThreads == 32 || blocks == 1;
  if (alone && at == 0) write_scores<T>(p, row, sums);

  if (p.top > 0) {
    const float normalizer = normalizer_of(sums);  // of the row, where the block has all of it
    const auto found = [&](int r, uint64_t key) {
      if (alone)
        write_top(p, row, r, key, normalizer);
      else
        sh.top[r] = key;
    };
    const int count = int(sh.count);
    if (count <= G::kRoom) {
      if (!alone && at >= count && at < p.top) sh.top[at] = 0;  // a part of fewer logits
      for (int i = at; i < count; i += kThreads) {
        const uint64_t key = sh.keys[i];
        int above = 0;
        for (int k = 0; k < count; ++k) above += sh.keys[k] > key;
        if (above < p.top) found(above, key);
      }
    } else {
      uint64_t last = ~uint64_t(0);
      G::sync();  // the keys' room is free
      for (int n = 0; n < p.top; ++n) {
        uint64_t best = 0;
        for (int from = begin; from < end; from += kTile) {
          if (!one_tile) load_tile(from);
#pragma unroll
          for (int r = 0; r < kVectors; ++r) {
            const int i = from + r * kThreads + at;
            if (i >= end) continue;
#pragma unroll
            for (int j = 0; j < kValues; ++j) {
              const int64_t place = grid.place(i) + j;
              const uint64_t key = key_of(word_value<T>(w[r], j), uint32_t(place));
              if (place >= 0 && place < p.v && key < last && key > best) best = key;
            }
          }
        }
        last = G::most(best, sh.keys);
        if (at == 0) found(n, last);
      }
    }
  }
  if (alone) return;

  // The cluster's first block joins the parts: their sums in order, and their alternatives by their ranks.
  if (at == 0) sh.of_block[0] = sums.m, sh.of_block[1] = sums.s, sh.of_block[2] = sums.w;
  cluster.sync();
  if (rank == 0) {
    Sums all{sums.m, 0.0f, 0.0f};
    for (int b = 1; b < blocks; ++b) all.m = larger(all.m, cluster.map_shared_rank(sh.of_block, b)[0]);
    for (int b = 0; b < blocks; ++b) {
      const float* const of = cluster.map_shared_rank(sh.of_block, b);
      const Sums one = moved(Sums{of[0], of[1], of[2]}, all.m);
      all.s += one.s, all.w += one.w;
    }
    if (at == 0) write_scores<T>(p, row, all);
    if (p.top > 0) {
      const int count = blocks * p.top;
      for (int i = at; i < count; i += kThreads) sh.keys[i] = cluster.map_shared_rank(sh.top, i / p.top)[i % p.top];
      __syncthreads();
      const float normalizer = normalizer_of(all);
      for (int i = at; i < count; i += kThreads) {
        const uint64_t key = sh.keys[i];
        int above = 0;
        for (int k = 0; k < count; ++k) above += sh.keys[k] > key;
        if (key && above < p.top) write_top(p, row, above, key, normalizer);
      }
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
};

// What a row's gradients have in common.
struct RowGrad {
  float g, h, normalizer, entropy;
  int64_t action;
  RLENV_D RowGrad(const ScoresGrad& p, int64_t row) {
    action = action_of(p.actions, p.action_dtype, row);
    check_flag(action >= p.v, kCheckActionRange);
    g = p.grad_log_prob && action >= 0 ? __ldg(p.grad_log_prob + row) : 0.0f;
    if (action >= p.v) g = not_a_number();
    h = p.grad_entropy ? __ldg(p.grad_entropy + row) : 0.0f;
    normalizer = __ldg(p.normalizer + row), entropy = __ldg(p.entropy + row);
  }
  RLENV_D float at(float l, int64_t place) const {
    if (l == -infinity() || normalizer == -infinity()) return 0.0f;
    const float lp = larger(l - normalizer, kFar), prob = __expf(lp);
    return g * ((place == action ? 1.0f : 0.0f) - prob) - h * prob * (lp + entropy);
  }
};

RLENV_D void store_value(float* to, float x) { *to = x; }
RLENV_D void store_value(__nv_bfloat16* to, float x) { *to = __float2bfloat16_rn(x); }

// Rows of few actions: a thread an element.
constexpr int kFlat = 4;
template <typename T>
__global__ void __launch_bounds__(256) few_scores_grad_kernel(const __grid_constant__ ScoresGrad p) {
  const int64_t first = int64_t(blockIdx.x) * 256 * kFlat, row0 = first / p.v;
  const uint32_t in = uint32_t(first - row0 * p.v), v = uint32_t(p.v);
#pragma unroll
  for (int i = 0; i < kFlat; ++i) {
    const uint32_t off = in + threadIdx.x + 256 * i;
    const int64_t row = row0 + off / v;
    if (row >= p.m) return;
    const uint32_t j = off % v;
    const RowGrad grad(p, row);
    const bool open = !p.allowed || p.allowed[row * p.allowed_stride + j];
    const float l = open ? value_at(static_cast<const T*>(p.logits) + row * p.stride + j) : -infinity();
    store_value(static_cast<T*>(p.grad) + row * p.v + j, grad.at(l, j));
  }
}

// A warp a run of kRun vectors of a row of the gradient, on its 16-byte boundaries. With y = log2 p the gradient of what
// was not chosen is - p (g + h entropy + h ln 2 y): two values an instruction but for the power.
constexpr int kRun = 128;
template <typename T>
__global__ void __launch_bounds__(256) scores_grad_kernel(const __grid_constant__ ScoresGrad p, int64_t runs) {
  constexpr int kValues = Grid<T>::kValues, kVectors = kRun / 32;
  const int64_t warp = int64_t(blockIdx.x) * 8 + threadIdx.x / 32, row = warp / runs;
  if (row >= p.m) return;
  const int lane = threadIdx.x % 32, first = int(warp - row * runs) * kRun + lane;
  const T* const logits = static_cast<const T*>(p.logits) + row * p.stride;
  const uint8_t* const allowed = p.allowed ? p.allowed + row * p.allowed_stride : nullptr;
  T* const grad = static_cast<T*>(p.grad) + row * p.v;
  const Grid<T> to(grad, p.v), from(logits, p.v);
  const int vectors = int(to.vectors());
  uint32_t w[kVectors][4];
#pragma unroll
  for (int r = 0; r < kVectors; ++r) {
    const int i = first + 32 * r;
    if (i >= vectors) continue;
    if (to.skip == from.skip) {
      load_vector(from, allowed, i, w[r]);
    } else {
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        w[r][k] = 0;
#pragma unroll
        for (int h = 0; h < kValues / 4; ++h) {
          const int64_t place = to.place(i) + k * (kValues / 4) + h;
          const bool open = place >= 0 && place < p.v && (!allowed || allowed[place]);
          const uint32_t x = __float_as_uint(open ? value_at(logits + place) : -infinity());
          w[r][k] |= sizeof(T) == 4 ? x : x >> 16 << 16 * h;
        }
      }
    }
  }
  const RowGrad of(p, row);
  const bool none = of.normalizer == -infinity();
  const float base = none ? 0.0f : of.normalizer;
  const float a = none ? 0.0f : -(of.g + of.h * of.entropy), b = none ? 0.0f : -of.h * kLn2;
  const uint64_t minus_base = pair_of(-base, -base), a2 = pair_of(a, a), b2 = pair_of(b, b);
#pragma unroll
  for (int r = 0; r < kVectors; ++r) {
    const int i = first + 32 * r;
    if (i >= vectors) continue;
    const int64_t j0 = to.place(i);
    float x[kValues];
#pragma unroll
    for (int k = 0; k < kValues / 2; ++k) {
      const uint64_t y = powers_of(word_pair<T>(w[r], k), minus_base);
      const float2 q = values_of(y);
      const uint64_t prob = pair_of(exp2_fast(q.x), exp2_fast(q.y));
      const float2 v = values_of(multiply_pairs(prob, multiply_add_pairs(b2, y, a2)));
      x[2 * k] = v.x, x[2 * k + 1] = v.y;
    }
    const int64_t chosen = of.action - j0;
    if (chosen >= 0 && chosen < kValues && !none) {
#pragma unroll
      for (int j = 0; j < kValues; ++j)
        if (j == chosen && word_value<T>(w[r], j) != -infinity()) x[j] += of.g;
    }
    if (j0 >= 0 && j0 + kValues <= p.v) {
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

template <typename T, int kLanes>
int few_scores(const Scores& p, cudaStream_t s) {
  few_scores_kernel<T, kLanes><<<unsigned((p.m * kLanes + 255) / 256), 256, 0, s>>>(p);
  return launch_status();
}
template <typename T, int kThreads, int kVectors>
int scores(const Scores& p, int blocks, cudaStream_t s) {
  using G = Team<kThreads>;
  cudaLaunchConfig_t config{};
  config.gridDim = dim3(unsigned(kThreads == 32 ? (p.m + G::kRows - 1) / G::kRows : p.m * blocks));
  config.blockDim = dim3(G::kBlock);
  config.stream = s;
  cudaLaunchAttribute cluster{};
  cluster.id = cudaLaunchAttributeClusterDimension;
  cluster.val.clusterDim.x = unsigned(blocks), cluster.val.clusterDim.y = cluster.val.clusterDim.z = 1;
  config.attrs = &cluster, config.numAttrs = blocks > 1 ? 1 : 0;
  const cudaError_t e = cudaLaunchKernelEx(&config, scores_kernel<T, kThreads, kVectors>, p);
  return e == cudaSuccess ? launch_status() : int(e);
}

template <typename T>
int scores_of(const Scores& p, cudaStream_t s) {
  constexpr int kValues = Grid<T>::kValues;
  if (p.v <= kEach) return few_scores<T, 1>(p, s);
  if (p.v <= 2 * kEach) return few_scores<T, 2>(p, s);
  if (p.v <= 4 * kEach) return few_scores<T, 4>(p, s);
  if (p.v <= 8 * kEach) return few_scores<T, 8>(p, s);
  if (p.v <= 32 * kEach) return few_scores<T, 32>(p, s);
  const bool on_lines = at_multiple(p.logits, 16) && p.stride % kValues == 0;
  const int64_t vectors = (p.v + (on_lines ? kValues - 1 : 2 * kValues - 2)) / kValues;  // at most
  if (vectors <= 64) return scores<T, 32, 2>(p, 1, s);
  if (vectors <= 128) return scores<T, 32, 4>(p, 1, s);
  if (vectors <= 256) return scores<T, 32, 8>(p, 1, s);
  if (vectors <= 1024) return scores<T, 128, 8>(p, 1, s);
  // A part of a row for each block of a cluster: until it fits into the registers, and while blocks are few and a part
  // has a vector for each thread.
  int blocks = 1;
  while (blocks < 8 && (vectors > 512 * 8 * blocks || (p.m * blocks < 296 && vectors > 512 * blocks))) blocks *= 2;
  if (vectors <= 512 * 2 * blocks) return scores<T, 512, 2>(p, blocks, s);
  if (vectors <= 512 * 4 * blocks) return scores<T, 512, 4>(p, blocks, s);
  return scores<T, 512, 8>(p, blocks, s);
}

template <typename T>
int scores_grad_of(const ScoresGrad& p, cudaStream_t s) {
  constexpr int kValues = Grid<T>::kValues;
  if (p.v < 64) {
    few_scores_grad_kernel<T><<<unsigned((p.m * p.v + 256 * kFlat - 1) / (256 * kFlat)), 256, 0, s>>>(p);
  } else {
    const int64_t vectors = (p.v + 2 * kValues - 2) / kValues, runs = (vectors + kRun - 1) / kRun;
    scores_grad_kernel<T><<<unsigned((p.m * runs + 7) / 8), 256, 0, s>>>(p, runs);
  }
  return launch_status();
}

bool scores_sizes(int dtype, int64_t m, int64_t v, int64_t stride, int action_dtype, int64_t allowed_stride) {
  return (dtype == RLENV_F32 || dtype == RLENV_BF16) && m >= 0 && v >= 1 && v < (int64_t(1) << 31) &&
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
  using namespace rlenv;
  if (!scores_sizes(dtype, m, v, stride, action_dtype, allowed_stride) || top < 0 || top > kMostTop || top > v)
    return RLENV_EINVAL;
  if (m == 0) return RLENV_OK;
  if (!logits || !actions || !log_prob || !entropy || !normalizer || (top > 0 && (!top_actions || !top_log_probs)))
    return RLENV_EINVAL;
  if (!at_multiple(logits, dtype == RLENV_F32 ? 4 : 2) || !at_multiple(actions, action_size(action_dtype)) ||
      !at_multiple(log_prob, 4) || !at_multiple(entropy, 4) || !at_multiple(normalizer, 4) || !at_multiple(top_actions, 8) ||
      !at_multiple(top_log_probs, 4))
    return RLENV_EINVAL;
  const Scores p{m, v, logits, stride, actions, action_dtype, allowed, allowed_stride, log_prob, entropy, normalizer,
                 top, top_actions, top_log_probs};
  return dtype == RLENV_F32 ? scores_of<float>(p, as_stream(stream)) : scores_of<__nv_bfloat16>(p, as_stream(stream));
}

int rlenv_log_probs_backward(int dtype, int64_t m, int64_t v, const float* grad_log_prob, const float* grad_entropy,
                             const void* logits, int64_t stride, const void* actions, int action_dtype,
                             const float* normalizer, const float* entropy, const uint8_t* allowed, int64_t allowed_stride,
                             void* grad, void* stream) {
  using namespace rlenv;
  if (!scores_sizes(dtype, m, v, stride, action_dtype, allowed_stride)) return RLENV_EINVAL;
  if (m == 0) return RLENV_OK;
  const int size = dtype == RLENV_F32 ? 4 : 2;
  if (!logits || !actions || !normalizer || !entropy || !grad || !at_multiple(logits, size) || !at_multiple(grad, size) ||
      !at_multiple(actions, action_size(action_dtype)) || !at_multiple(normalizer, 4) || !at_multiple(entropy, 4) ||
      !at_multiple(grad_log_prob, 4) || !at_multiple(grad_entropy, 4))
    return RLENV_EINVAL;
  const ScoresGrad p{m, v, grad_log_prob, grad_entropy, logits, stride, actions, action_dtype, normalizer, entropy, allowed,
                     allowed_stride, grad};
  return dtype == RLENV_F32 ? scores_grad_of<float>(p, as_stream(stream))
                            : scores_grad_of<__nv_bfloat16>(p, as_stream(stream));
}

}  // extern "C"
