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
// Bound by memory: 8 bytes of parameter and the gradient, and 16 (32-bit moments) or 4 (8-bit)
// bytes of moments an element.
#include <cuda_bf16.h>
#include <math.h>

#include "common.cuh"

namespace rlenv {
namespace {

constexpr int kStateBlock = 256;
constexpr int kAdamThreads = 256;
constexpr int kAdamTensors = 96;  // tensors per launch: their table travels in the launch's parameters

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

RLENV_D float load_grad(const float* g, int64_t i) { return __ldg(g + i); }
RLENV_D float load_grad(const __nv_bfloat16* g, int64_t i) { return __bfloat162float(g[i]); }
RLENV_D void load_grad4(const float* g, int64_t i, float o[4]) {
  const float4 x = __ldg(reinterpret_cast<const float4*>(g + i));
  o[0] = x.x, o[1] = x.y, o[2] = x.z, o[3] = x.w;
}
RLENV_D void load_grad4(const __nv_bfloat16* g, int64_t i, float o[4]) {
  const uint2 x = __ldg(reinterpret_cast<const uint2*>(g + i));
  o[0] = __uint_as_float(x.x << 16), o[1] = __uint_as_float(x.x & 0xffff0000u);
  o[2] = __uint_as_float(x.y << 16), o[3] = __uint_as_float(x.y & 0xffff0000u);
}

RLENV_D float sqrt_approx(float x) {  // within an ulp; only the update passes through it
  float r;
  asm("sqrt.approx.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

constexpr uint32_t kInfBits = 0x7f800000u;

// E exponent bits: see the top of the file.
template <int E>
RLENV_D float decode(uint32_t c, uint32_t e) {
  constexpr uint32_t kTop = (1u << (E + 3)) - 1;
  const uint32_t mag = c & kTop;
  const uint32_t bits = (mag + 8u * (e - ((1u << E) - 1u))) << 20;
  float x = mag == 0 ? 0.0f : mag == kTop ? __uint_as_float(0x7fffffffu) : __uint_as_float(bits);
  return E == 4 && (c & 128u) ? -x : x;
}

// The block's shared exponent from the bits of its largest finite magnitude.
RLENV_D uint32_t block_exponent(uint32_t bits) {
  const uint32_t e = (bits + 0x1fffffu) >> 23;
  return e < 32u ? 32u : e;
}

template <int E>
RLENV_D uint32_t encode(float x, uint32_t e, uint32_t rand16) {
  constexpr int kTop = (1 << (E + 3)) - 1;
  const uint32_t bits = __float_as_uint(x) & 0x7fffffffu;
  int c = int((bits + (rand16 << 4)) >> 20) - 8 * (int(e) - ((1 << E) - 1));
  c = max(c, E == 5 && bits > 0 ? 1 : 0);
  if (bits >= kInfBits) c = kTop;
  return uint32_t(c) | (E == 4 ? (__float_as_uint(x) >> 31) << 7 : 0u);
}

// A warp owns a state block: lane l elements 4 l .. 4 l + 3 and 128 + 4 l .. + 3.
template <typename G, bool kEight>
__global__ void __launch_bounds__(kAdamThreads) adamw_kernel(const __grid_constant__ AdamArgs a) {
  const uint32_t local = blockIdx.x * (kAdamThreads / 32) + (threadIdx.x >> 5);
  if (local >= a.blocks) return;
  const uint32_t block = a.t[0].first + local;
  const int lane = threadIdx.x & 31;
  int lo = 0, hi = a.count - 1;  // the last tensor that starts at or before the block
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (a.t[mid].first <= block) lo = mid; else hi = mid - 1;
  }
  const AdamTensor t = a.t[lo];
  const G* grad = static_cast<const G*>(t.g);
  const int64_t base = int64_t(block - t.first) * kStateBlock;  // in the tensor
  const int64_t flat = int64_t(block) * kStateBlock;            // in the moments
  const float gs = a.grad_scale ? __ldg(a.grad_scale) : 1.0f;

  float p[8], g[8], m[8], v[8];
  uint32_t em = 0, ev = 0;
  if constexpr (kEight) em = a.m_exp[block], ev = a.v_exp[block];
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    const int64_t i = base + 128 * u + 4 * lane;
    if (t.wide && i + 4 <= t.n) {
      const float4 x = *reinterpret_cast<const float4*>(t.p + i);
      p[4 * u] = x.x, p[4 * u + 1] = x.y, p[4 * u + 2] = x.z, p[4 * u + 3] = x.w;
      load_grad4(grad, i, g + 4 * u);
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const bool in = i + j < t.n;
        p[4 * u + j] = in ? t.p[i + j] : 0.0f;
        g[4 * u + j] = in ? load_grad(grad, i + j) : 0.0f;
      }
    }
    const int64_t f = flat + 128 * u + 4 * lane;
    if constexpr (kEight) {
      const uint32_t cm = *reinterpret_cast<const uint32_t*>(static_cast<const uint8_t*>(a.m) + f);
      const uint32_t cv = *reinterpret_cast<const uint32_t*>(static_cast<const uint8_t*>(a.v) + f);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        m[4 * u + j] = decode<4>((cm >> (8 * j)) & 255u, em);
        v[4 * u + j] = decode<5>((cv >> (8 * j)) & 255u, ev);
      }
    } else {
      const float4 x = *reinterpret_cast<const float4*>(static_cast<const float*>(a.m) + f);
      const float4 y = *reinterpret_cast<const float4*>(static_cast<const float*>(a.v) + f);
      m[4 * u] = x.x, m[4 * u + 1] = x.y, m[4 * u + 2] = x.z, m[4 * u + 3] = x.w;
      v[4 * u] = y.x, v[4 * u + 1] = y.y, v[4 * u + 2] = y.z, v[4 * u + 3] = y.w;
    }
  }
  uint32_t top_m = 0, top_v = 0;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const float x = __fmul_rn(g[j], gs);
    m[j] = __fadd_rn(__fmul_rn(m[j], a.b1), __fmul_rn(x, a.c1));
    v[j] = __fadd_rn(__fmul_rn(v[j], a.b2), __fmul_rn(__fmul_rn(x, x), a.c2));
    const float denom = sqrt_approx(v[j]) * a.root + a.eps;
    p[j] = __fsub_rn(__fmul_rn(p[j], a.keep), __fdividef(m[j] * a.rate, denom));
    if constexpr (kEight) {
      const uint32_t bm = __float_as_uint(m[j]) & 0x7fffffffu, bv = __float_as_uint(v[j]);
      if (bm < kInfBits) top_m = max(top_m, bm);
      if (bv < kInfBits) top_v = max(top_v, bv);
    }
  }
  if constexpr (kEight) {
    em = block_exponent(__reduce_max_sync(0xffffffffu, top_m));
    ev = block_exponent(__reduce_max_sync(0xffffffffu, top_v));
    if (lane == 0) a.m_exp[block] = uint8_t(em), a.v_exp[block] = uint8_t(ev);
  }
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    const int64_t i = base + 128 * u + 4 * lane;
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
    const int64_t f = flat + 128 * u + 4 * lane;
    if constexpr (kEight) {
      uint32_t cm = 0, cv = 0;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint32_t r = pcg_hash(uint32_t(f + j) ^ a.key);
        cm |= encode<4>(m[4 * u + j], em, r & 0xffffu) << (8 * j);
        cv |= encode<5>(v[4 * u + j], ev, r >> 16) << (8 * j);
      }
      *reinterpret_cast<uint32_t*>(static_cast<uint8_t*>(a.m) + f) = cm;
      *reinterpret_cast<uint32_t*>(static_cast<uint8_t*>(a.v) + f) = cv;
    } else {
      *reinterpret_cast<float4*>(static_cast<float*>(a.m) + f) =
          make_float4(m[4 * u], m[4 * u + 1], m[4 * u + 2], m[4 * u + 3]);
      *reinterpret_cast<float4*>(static_cast<float*>(a.v) + f) =
          make_float4(v[4 * u], v[4 * u + 1], v[4 * u + 2], v[4 * u + 3]);
    }
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
  const uint32_t em = __ldg(m_exp + i / (kStateBlock / 4)), ev = __ldg(v_exp + i / (kStateBlock / 4));
  m_out[i] = make_float4(decode<4>(cm & 255u, em), decode<4>((cm >> 8) & 255u, em), decode<4>((cm >> 16) & 255u, em),
                         decode<4>(cm >> 24, em));
  v_out[i] = make_float4(decode<5>(cv & 255u, ev), decode<5>((cv >> 8) & 255u, ev), decode<5>((cv >> 16) & 255u, ev),
                         decode<5>(cv >> 24, ev));
}

bool on_boundary(const void* p, int bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }

template <typename G, bool kEight>
int adamw_launch(const AdamArgs& a, cudaStream_t stream) {
  const unsigned grid = (a.blocks + kAdamThreads / 32 - 1) / (kAdamThreads / 32);
  adamw_kernel<G, kEight><<<grid, kAdamThreads, 0, stream>>>(a);
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
  if (!params || !grads || !sizes || !m || !v || (state_bits == 8 && (!m_exp || !v_exp))) return RLENV_EINVAL;
  if (!on_boundary(m, state_bits == 8 ? 4 : 16) || !on_boundary(v, state_bits == 8 ? 4 : 16)) return RLENV_EINVAL;
  int64_t total = 0;
  for (int64_t i = 0; i < tensors; ++i) {
    if (sizes[i] < 0 || sizes[i] > (int64_t(1) << 40)) return RLENV_EINVAL;
    if (sizes[i] > 0 && (!params[i] || !grads[i])) return RLENV_EINVAL;
    total += (sizes[i] + kStateBlock - 1) / kStateBlock;
    if (total > (int64_t(1) << 32) / kStateBlock) return RLENV_EINVAL;  // places are hashed as 32-bit words
  }
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
