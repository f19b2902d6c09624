// One AdamW step over many tensors (Loshchilov & Hutter, "Decoupled weight decay
// regularization", 2019), the moments in 32 bits or in 8:
//     m <- b1 m + (1 - b1) g,   v <- b2 v + (1 - b2) g^2,
//     p <- p (1 - lr wd) - lr (m / (1 - b1^t)) / (sqrt(v / (1 - b2^t)) + eps).
// Parameters are float32; gradients float32 or bfloat16; an optional bfloat16 copy of each
// parameter is written in the same pass. The moments of all tensors are two flat arrays in
// which each tensor starts at a multiple of kStateBlock elements.
//
// Moments in 8 bits. The kStateBlock elements of a block share an exponent e (a byte), that
// of their largest magnitude, one up where its mantissa is above 1.75. An element's code c > 0
// stands for the float whose bits are (c + 8 (e - 2^E + 1)) << 20: three mantissa bits and E
// bits of exponent counted down from e (E = 4 and a sign for m, E = 5 for v, whose range is
// the square of the gradients'); 0 stands for zero and the largest code for NaN, so that one
// element's infinity or NaN leaves its neighbours as they are. A step changes v by as little as
// a thousandth, far less than half of a code's 6 to 12%: rounding to nearest would never move it.
// So rounding is stochastic: 16 random bits are added below the last kept bit, a hash of (seed,
// step, place), which keeps the moments right on average. v > 0 never rounds to zero (a zero
// would leave eps alone in the denominator). All arithmetic on the moments is in 32 bits, each
// product and sum rounded on its own (no fused multiply-add), so that codes are reproducible.
//
// Bound by memory with 32-bit moments: 8 bytes of parameter, the gradient and 16 bytes of moments an element
// (60 M elements with bfloat16 gradients and copies 277 us, 6.1 TB/s). With 8-bit ones, 4 bytes of moments, by
// instructions: 213 us, 4.5 TB/s.
#include <cuda_bf16.h>
#include <math.h>

#include "common.cuh"

namespace rlenv {
namespace {

constexpr int kStateBlock = 256;
constexpr int kAdamThreads = 256;
constexpr int kAdamTensors = 96;    // tensors per launch: their table travels in the launch's parameters

// Blocks of threads on an SM: 8-bit moments, bound by instructions, want as many as their registers allow (213 us
// against 217 with three, 228 with two, for 60 M parameters); 32-bit ones, bound by memory, two, with more in
// flight each (277 us against 289 with three, 314 with four).
constexpr int kPerSm[2] = {2, 4}, kSms = 148;  // 32 bits, 8 bits

struct AdamTensor {
  float* p;
  const void* g;
  __nv_bfloat16* copy;
  int64_t n;
  uint32_t first;  // first state block
  uint32_t wide;   // p, g and copy on the boundaries of four-element accesses
};

struct AdamArgs {
  float b1, c1, b2, c2;      // c = 1 - b
  float rate, root, eps;     // lr / (1 - b1^t), 1 / sqrt(1 - b2^t)
  float keep;                // 1 - lr wd
  uint32_t key;
  uint32_t blocks;           // state blocks of this launch, from the first tensor's
  int count;
  const float* grad_scale;
  void *m, *v;
  uint8_t *m_exp, *v_exp;
  AdamTensor t[kAdamTensors];
};

// Four gradients as they are stored.
template <typename G>
struct FourGrads;
template <>
struct FourGrads<float> {
  float4 raw;
  RLENV_D void load(const float* g, int64_t i) { raw = __ldg(reinterpret_cast<const float4*>(g + i)); }
  RLENV_D void load(const float* g, int64_t i, int64_t n) {
    raw = make_float4(i < n ? g[i] : 0.0f, i + 1 < n ? g[i + 1] : 0.0f, i + 2 < n ? g[i + 2] : 0.0f,
                      i + 3 < n ? g[i + 3] : 0.0f);
  }
  RLENV_D float4 values() const { return raw; }
};
template <>
struct FourGrads<__nv_bfloat16> {
  uint2 raw;
  RLENV_D void load(const __nv_bfloat16* g, int64_t i) { raw = __ldg(reinterpret_cast<const uint2*>(g + i)); }
  RLENV_D void load(const __nv_bfloat16* from, int64_t i, int64_t n) {
    const unsigned short* g = reinterpret_cast<const unsigned short*>(from);
    raw = make_uint2((i < n ? g[i] : 0u) | (i + 1 < n ? uint32_t(g[i + 1]) << 16 : 0u),
                     (i + 2 < n ? g[i + 2] : 0u) | (i + 3 < n ? uint32_t(g[i + 3]) << 16 : 0u));
  }
  RLENV_D float4 values() const {
    return make_float4(__uint_as_float(raw.x << 16), __uint_as_float(raw.x & 0xffff0000u),
                       __uint_as_float(raw.y << 16), __uint_as_float(raw.y & 0xffff0000u));
  }
};

// The update's root and quotient from the special function unit, within 2 ulp; no moment passes through
// them. Values below 2^-126 count as zero, so that sqrt(v) is off by up to 2^-63: nothing beside an epsilon of
// 2^-40 and more (times `root`). A smaller one, zero among them, takes the exactly rounded functions (kExact).
RLENV_D float sqrt_approx(float x) {
  float r;
  asm("sqrt.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
RLENV_D float quotient_approx(float x, float y) {
  float r;
  asm("div.approx.ftz.f32 %0, %1, %2;" : "=f"(r) : "f"(x), "f"(y));
  return r;
}

constexpr uint32_t kInfBits = 0x7f800000u, kNanBits = 0x7fffffffu, kCodeBit = 1u << 20;

// E exponent bits (see the top of the file): a code's value is the float whose bits are its magnitude << 20
// plus base<E>(e), so that both ways are an addition.
template <int E>
RLENV_D uint32_t base(uint32_t e) { return (8u * (e - ((1u << E) - 1u))) << 20; }

template <int E, bool kTops>
RLENV_D float decode(uint32_t c, uint32_t from) {
  constexpr uint32_t kTop = (1u << (E + 3)) - 1;
  const uint32_t mag = c & kTop;
  uint32_t bits = mag == 0 ? 0u : (mag << 20) + from;
  if (kTops && mag == kTop) bits = kNanBits;
  return __uint_as_float(E == 4 ? bits | (c & 128u) << 24 : bits);
}
// Whether any of four codes is the largest, NaN's.
template <int E>
RLENV_D uint32_t any_top(uint32_t c) {
  const uint32_t sevens = (c & 0x7f7f7f7fu) + 0x01010101u;  // the high bit of a byte whose low seven are ones
  return (E == 4 ? sevens : c & sevens) & 0x80808080u;
}

// The block's shared exponent from the bits of its largest finite magnitude.
RLENV_D uint32_t block_exponent(uint32_t bits) {
  const uint32_t e = (bits + 0x1fffffu) >> 23;
  return e < 32u ? 32u : e;
}

// The code in the top byte. rand4: the random bits at 4..19. kSpecial: x may be infinite or NaN.
template <int E, bool kSpecial>
RLENV_D uint32_t encode_high(float x, uint32_t from, uint32_t rand4) {
  constexpr uint32_t kTop = (1u << (E + 3)) - 1;
  const uint32_t bits = __float_as_uint(x) & 0x7fffffffu;
  // negative where x is below the block's range; v > 0 has at least code 1
  int place = max(int(bits + rand4 - from), E == 5 && bits > 0 ? int(kCodeBit) : 0);
  if (kSpecial && bits >= kInfBits) place = int(kTop << 20);
  return (uint32_t(place) << 4 & (E == 4 ? 0x7f000000u : 0xff000000u)) | (E == 4 ? __float_as_uint(x) & 0x80000000u : 0u);
}
RLENV_D uint32_t top_bytes(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  return __byte_perm(__byte_perm(a, b, 0x0073), __byte_perm(c, d, 0x0073), 0x5410);
}

template <bool kSpecial>
RLENV_D void encode_four(const float* m, const float* v, uint32_t place, uint32_t from_m, uint32_t from_v,
                         uint32_t* cm, uint32_t* cv) {
  uint32_t a[4], b[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const uint32_t r = pcg_hash(place ^ j);
    a[j] = encode_high<4, kSpecial>(m[j], from_m, r << 4 & 0xffff0u);
    b[j] = encode_high<5, kSpecial>(v[j], from_v, r >> 12 & 0xffff0u);
  }
  *cm = top_bytes(a[0], a[1], a[2], a[3]);
  *cv = top_bytes(b[0], b[1], b[2], b[3]);
}

// What a lane reads of a state block: elements 4 l .. 4 l + 3 and 128 + 4 l .. + 3.
template <typename G, bool kEight>
struct Elements {
  float4 p[2], m[kEight ? 1 : 2], v[kEight ? 1 : 2];
  FourGrads<G> g[2];
  uint32_t cm[2], cv[2], em, ev;

  RLENV_D void load(const AdamArgs& a, const AdamTensor& t, uint32_t block, int lane) {
    const int64_t in = int64_t(block - t.first) * kStateBlock + 4 * lane;  // in the tensor
    const int64_t flat = int64_t(block) * kStateBlock + 4 * lane;          // in the moments
    const G* grad = static_cast<const G*>(t.g);
    if constexpr (kEight) em = a.m_exp[block], ev = a.v_exp[block];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int64_t i = in + 128 * u, f = flat + 128 * u;
      if constexpr (kEight) {
        cm[u] = *reinterpret_cast<const uint32_t*>(static_cast<const uint8_t*>(a.m) + f);
        cv[u] = *reinterpret_cast<const uint32_t*>(static_cast<const uint8_t*>(a.v) + f);
      } else {
        m[u] = *reinterpret_cast<const float4*>(static_cast<const float*>(a.m) + f);
        v[u] = *reinterpret_cast<const float4*>(static_cast<const float*>(a.v) + f);
      }
      if (t.wide && i + 4 <= t.n) {
        p[u] = *reinterpret_cast<const float4*>(t.p + i);
        g[u].load(grad, i);
      } else {
        p[u] = make_float4(i < t.n ? t.p[i] : 0.0f, i + 1 < t.n ? t.p[i + 1] : 0.0f, i + 2 < t.n ? t.p[i + 2] : 0.0f,
                           i + 3 < t.n ? t.p[i + 3] : 0.0f);
        g[u].load(grad, i, t.n);
      }
    }
  }
};

RLENV_D void unpack(const float4& x, float* to) { to[0] = x.x, to[1] = x.y, to[2] = x.z, to[3] = x.w; }

// A warp takes every stride-th state block and reads one ahead: a block's arithmetic, some 80 instructions an
// element with 8-bit moments, runs under the next one's loads.
template <typename G, bool kEight, bool kExact>
__global__ void __launch_bounds__(kAdamThreads, kPerSm[kEight]) adamw_kernel(const __grid_constant__ AdamArgs a) {
  const int lane = threadIdx.x & 31;
  const uint32_t stride = gridDim.x * (kAdamThreads / 32), end = a.t[0].first + a.blocks;
  uint32_t block = a.t[0].first + blockIdx.x * (kAdamThreads / 32) + (threadIdx.x >> 5);
  if (block >= end) return;
  int at = 0, hi = a.count - 1;  // the last tensor that starts at or before the block
  while (at < hi) {
    const int mid = (at + hi + 1) >> 1;
    if (a.t[mid].first <= block) at = mid; else hi = mid - 1;
  }
  const float gs = a.grad_scale ? __ldg(a.grad_scale) : 1.0f;
  Elements<G, kEight> ahead;
  ahead.load(a, a.t[at], block, lane);
  while (true) {
    const Elements<G, kEight> x = ahead;
    const AdamTensor& t = a.t[at];
    const uint32_t next = block + stride;
    int next_at = at;
    if (next < end) {
      while (next_at + 1 < a.count && a.t[next_at + 1].first <= next) ++next_at;
      ahead.load(a, a.t[next_at], next, lane);
    }
    const int64_t in = int64_t(block - t.first) * kStateBlock + 4 * lane, flat = int64_t(block) * kStateBlock + 4 * lane;
    float p[8], g[8], m[8], v[8];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      unpack(x.p[u], p + 4 * u);
      unpack(x.g[u].values(), g + 4 * u);
      if constexpr (!kEight) unpack(x.m[u], m + 4 * u), unpack(x.v[u], v + 4 * u);
    }
    if constexpr (kEight) {
      const uint32_t from_m = base<4>(x.em), from_v = base<5>(x.ev);
      const uint32_t tops = any_top<4>(x.cm[0]) | any_top<4>(x.cm[1]) | any_top<5>(x.cv[0]) | any_top<5>(x.cv[1]);
      if (__any_sync(0xffffffffu, tops != 0)) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          m[j] = decode<4, true>(x.cm[j / 4] >> (8 * (j % 4)) & 255u, from_m);
          v[j] = decode<5, true>(x.cv[j / 4] >> (8 * (j % 4)) & 255u, from_v);
        }
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          m[j] = decode<4, false>(x.cm[j / 4] >> (8 * (j % 4)) & 255u, from_m);
          v[j] = decode<5, false>(x.cv[j / 4] >> (8 * (j % 4)) & 255u, from_v);
        }
      }
    }
    uint32_t top_m = 0, top_v = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float y = __fmul_rn(g[j], gs);
      m[j] = __fadd_rn(__fmul_rn(m[j], a.b1), __fmul_rn(y, a.c1));
      v[j] = __fadd_rn(__fmul_rn(v[j], a.b2), __fmul_rn(__fmul_rn(y, y), a.c2));
      const float denom = fmaf(kExact ? __fsqrt_rn(v[j]) : sqrt_approx(v[j]), a.root, a.eps), top = m[j] * a.rate;
      p[j] = __fsub_rn(__fmul_rn(p[j], a.keep), kExact ? __fdiv_rn(top, denom) : quotient_approx(top, denom));
      if constexpr (kEight) {
        top_m = max(top_m, __float_as_uint(m[j]) & 0x7fffffffu);
        top_v = max(top_v, __float_as_uint(v[j]) & 0x7fffffffu);
      }
    }
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int64_t i = in + 128 * u;
      if (t.wide && i + 4 <= t.n) {
        *reinterpret_cast<float4*>(t.p + i) = make_float4(p[4 * u], p[4 * u + 1], p[4 * u + 2], p[4 * u + 3]);
        if (t.copy) {
          const __nv_bfloat162 lo2 = __floats2bfloat162_rn(p[4 * u], p[4 * u + 1]);
          const __nv_bfloat162 hi2 = __floats2bfloat162_rn(p[4 * u + 2], p[4 * u + 3]);
          *reinterpret_cast<uint2*>(t.copy + i) =
              make_uint2(*reinterpret_cast<const uint32_t*>(&lo2), *reinterpret_cast<const uint32_t*>(&hi2));
        }
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (i + j < t.n) {
            t.p[i + j] = p[4 * u + j];
            if (t.copy) t.copy[i + j] = __float2bfloat16_rn(p[4 * u + j]);
          }
      }
    }
    if constexpr (kEight) {
      top_m = __reduce_max_sync(0xffffffffu, top_m);
      top_v = __reduce_max_sync(0xffffffffu, top_v);
      const bool special = max(top_m, top_v) >= kInfBits;
      if (special) {  // the largest finite ones
        top_m = top_v = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const uint32_t bm = __float_as_uint(m[j]) & 0x7fffffffu, bv = __float_as_uint(v[j]) & 0x7fffffffu;
          if (bm < kInfBits) top_m = max(top_m, bm);
          if (bv < kInfBits) top_v = max(top_v, bv);
        }
        top_m = __reduce_max_sync(0xffffffffu, top_m);
        top_v = __reduce_max_sync(0xffffffffu, top_v);
      }
      const uint32_t em = block_exponent(top_m), ev = block_exponent(top_v);
      if (lane == 0) a.m_exp[block] = uint8_t(em), a.v_exp[block] = uint8_t(ev);
      const uint32_t from_m = base<4>(em), from_v = base<5>(ev);
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const uint32_t place = uint32_t(flat + 128 * u) ^ a.key;  // a multiple of four before the key
        uint32_t cm, cv;
        if (special) encode_four<true>(m + 4 * u, v + 4 * u, place, from_m, from_v, &cm, &cv);
        else encode_four<false>(m + 4 * u, v + 4 * u, place, from_m, from_v, &cm, &cv);
        *reinterpret_cast<uint32_t*>(static_cast<uint8_t*>(a.m) + flat + 128 * u) = cm;
        *reinterpret_cast<uint32_t*>(static_cast<uint8_t*>(a.v) + flat + 128 * u) = cv;
      }
    } else {
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        *reinterpret_cast<float4*>(static_cast<float*>(a.m) + flat + 128 * u) =
            make_float4(m[4 * u], m[4 * u + 1], m[4 * u + 2], m[4 * u + 3]);
        *reinterpret_cast<float4*>(static_cast<float*>(a.v) + flat + 128 * u) =
            make_float4(v[4 * u], v[4 * u + 1], v[4 * u + 2], v[4 * u + 3]);
      }
    }
    if (next >= end) return;
    block = next, at = next_at;
  }
}

// The values that 8-bit moments stand for.
__global__ void __launch_bounds__(256)
moments_kernel(const uint32_t* __restrict__ m, const uint32_t* __restrict__ v, const uint8_t* __restrict__ m_exp,
               const uint8_t* __restrict__ v_exp, int64_t quads, float4* __restrict__ m_out,
               float4* __restrict__ v_out) {
  const int64_t i = int64_t(blockIdx.x) * 256 + threadIdx.x;
  if (i >= quads) return;
  const uint32_t cm = __ldg(m + i), cv = __ldg(v + i);
  const uint32_t em = base<4>(__ldg(m_exp + i / (kStateBlock / 4))), ev = base<5>(__ldg(v_exp + i / (kStateBlock / 4)));
  m_out[i] = make_float4(decode<4, true>(cm & 255u, em), decode<4, true>((cm >> 8) & 255u, em), decode<4, true>((cm >> 16) & 255u, em),
                         decode<4, true>(cm >> 24, em));
  v_out[i] = make_float4(decode<5, true>(cv & 255u, ev), decode<5, true>((cv >> 8) & 255u, ev), decode<5, true>((cv >> 16) & 255u, ev),
                         decode<5, true>(cv >> 24, ev));
}

bool on_boundary(const void* p, int bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }

template <typename G, bool kEight>
int adamw_launch(const AdamArgs& a, cudaStream_t stream) {
  constexpr uint32_t kWarps = kAdamThreads / 32, kMost = kSms * kPerSm[kEight];
  const uint32_t grid = (a.blocks + kWarps - 1) / kWarps < kMost ? (a.blocks + kWarps - 1) / kWarps : kMost;
  constexpr float kApproxEps = 0x1p-40f;
  if (a.eps >= kApproxEps * a.root) adamw_kernel<G, kEight, false><<<grid, kAdamThreads, 0, stream>>>(a);
  else adamw_kernel<G, kEight, true><<<grid, kAdamThreads, 0, stream>>>(a);
  return launch_status();
}

}  // namespace
}  // namespace rlenv

extern "C" {

int rlenv_adamw_step(int state_bits, int grad_dtype, int64_t tensors, float* const* params, const void* const* grads,
                     void* const* copies, const int64_t* sizes, void* m, void* v, uint8_t* m_exp, uint8_t* v_exp,
                     double lr, double beta1, double beta2, double eps, double weight_decay, const float* grad_scale,
                     int64_t step, uint32_t seed, void* stream) {
  using namespace rlenv;
  if ((state_bits != 8 && state_bits != 32) || (grad_dtype != RLENV_F32 && grad_dtype != RLENV_BF16)) return RLENV_EINVAL;
  if (tensors < 0 || step < 1 || !(beta1 >= 0.0 && beta1 < 1.0) || !(beta2 >= 0.0 && beta2 < 1.0) || !(eps >= 0.0))
    return RLENV_EINVAL;
  if (tensors == 0) return RLENV_OK;
  if (!params || !grads || !sizes) return RLENV_EINVAL;
  int64_t total = 0;
  for (int64_t i = 0; i < tensors; ++i) {
    if (sizes[i] < 0 || sizes[i] > (int64_t(1) << 40)) return RLENV_EINVAL;
    if (sizes[i] > 0 && (!params[i] || !grads[i])) return RLENV_EINVAL;
    total += (sizes[i] + kStateBlock - 1) / kStateBlock;
    if (total > (int64_t(1) << 32) / kStateBlock) return RLENV_EINVAL;  // places are hashed as 32-bit words
  }
  if (total == 0) return RLENV_OK;  // moments of no elements may be NULL
  if (!m || !v || (state_bits == 8 && (!m_exp || !v_exp))) return RLENV_EINVAL;
  if (!on_boundary(m, state_bits == 8 ? 4 : 16) || !on_boundary(v, state_bits == 8 ? 4 : 16)) return RLENV_EINVAL;
  AdamArgs a;
  a.b1 = float(beta1), a.c1 = float(1.0 - beta1), a.b2 = float(beta2), a.c2 = float(1.0 - beta2);
  a.rate = float(lr / (1.0 - pow(beta1, double(step))));
  a.root = float(1.0 / sqrt(1.0 - pow(beta2, double(step))));
  a.eps = float(eps), a.keep = float(1.0 - lr * weight_decay);
  a.key = pcg_hash(seed ^ uint32_t(uint64_t(step) * 0x9E3779B9u));
  a.grad_scale = grad_scale, a.m = m, a.v = v, a.m_exp = m_exp, a.v_exp = v_exp;
  const int grad_size = grad_dtype == RLENV_F32 ? 4 : 2;
  uint32_t first = 0;
  for (int64_t i = 0; i < tensors;) {
    a.count = 0, a.blocks = 0;
    for (; i < tensors && a.count < kAdamTensors; ++i) {
      if (sizes[i] == 0) continue;
      AdamTensor& t = a.t[a.count++];
      t.p = params[i], t.g = grads[i], t.n = sizes[i], t.first = first;
      t.copy = copies ? static_cast<__nv_bfloat16*>(copies[i]) : nullptr;
      t.wide = on_boundary(t.p, 16) && on_boundary(t.g, 4 * grad_size) && on_boundary(t.copy, 8);
      const uint32_t blocks = uint32_t((sizes[i] + kStateBlock - 1) / kStateBlock);
      first += blocks, a.blocks += blocks;
    }
    if (a.count == 0) break;
    const cudaStream_t s = as_stream(stream);
    const int rc = state_bits == 8 ? (grad_dtype == RLENV_F32 ? adamw_launch<float, true>(a, s)
                                                              : adamw_launch<__nv_bfloat16, true>(a, s))
                                   : (grad_dtype == RLENV_F32 ? adamw_launch<float, false>(a, s)
                                                              : adamw_launch<__nv_bfloat16, false>(a, s));
    if (rc != RLENV_OK) return rc;
  }
  return RLENV_OK;
}

int rlenv_adamw_moments(int64_t blocks, const uint8_t* m, const uint8_t* v, const uint8_t* m_exp,
                        const uint8_t* v_exp, float* m_out, float* v_out, void* stream) {
  using namespace rlenv;
  if (blocks < 0 || blocks > (int64_t(1) << 32) / kStateBlock) return RLENV_EINVAL;
  if (blocks == 0) return RLENV_OK;
  if (!m || !v || !m_exp || !v_exp || !m_out || !v_out) return RLENV_EINVAL;
  if (!on_boundary(m, 4) || !on_boundary(v, 4) || !on_boundary(m_out, 16) || !on_boundary(v_out, 16))
    return RLENV_EINVAL;
  const int64_t quads = blocks * (kStateBlock / 4);
  moments_kernel<<<grid_for(quads, 256), 256, 0, as_stream(stream)>>>(
      reinterpret_cast<const uint32_t*>(m), reinterpret_cast<const uint32_t*>(v), m_exp, v_exp, quads,
      reinterpret_cast<float4*>(m_out), reinterpret_cast<float4*>(v_out));
  return launch_status();
}

}  // extern "C"
