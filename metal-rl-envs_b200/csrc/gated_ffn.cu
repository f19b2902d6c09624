// Gated feed-forward block: h = act(x Wg) * (x Wu) for x (M, K) and weights (K, F), and its
// gradient. With g = x Wg, u = x Wu and the gradient dh of h,
//     dg = dh u act'(g),   du = dh act(g),
//     dx = dg Wg' + du Wu',   dWg = x' dg,   dWu = x' du.
// The backward pass forms g and u again from x instead of keeping them: 2 M F values less to
// store and read, and no rounding of g and u to the inputs' type.
#include <cuda_bf16.h>

#include "common.cuh"

namespace rlenv {
namespace {

enum Activation { kSilu = 0, kGelu = 1 };

RLENV_D float load_f(const float* p, int64_t i) { return __ldg(p + i); }
RLENV_D float load_f(const __nv_bfloat16* p, int64_t i) { return __bfloat162float(p[i]); }
RLENV_D void store_f(float* p, int64_t i, float v) { p[i] = v; }
RLENV_D void store_f(__nv_bfloat16* p, int64_t i, float v) { p[i] = __float2bfloat16_rn(v); }

// act(g) and act'(g): silu g / (1 + e^-g), or gelu g Phi(g) with the exact normal distribution.
RLENV_D void activate(int act, float g, float* y, float* slope) {
  if (act == kSilu) {
    const float s = 1.0f / (1.0f + expf(-g));
    *y = g * s;
    *slope = s * (1.0f + g * (1.0f - s));
  } else {
    const float cdf = 0.5f * erfcf(-0.70710678f * g);
    *y = g * cdf;
    *slope = cdf + g * (0.39894228f * expf(-0.5f * g * g));
  }
}

constexpr int kTile = 64, kDepth = 16, kSimtThreads = 256;

// C(64 x 64 tile) += A B over one contraction of length k; A element (m, k) at a[m sam + k sak].
template <typename T>
struct Simt {
  float (*as)[kTile + 4];
  float (*bs)[kTile + 4];
  RLENV_D void run(const T* a, int64_t sam, int64_t sak, const T* b, int64_t sbk, int64_t sbn, int64_t m0, int64_t m,
                   int64_t n0, int64_t n, int64_t k, float acc[4][4]) const {
    const int tx = threadIdx.x % 16, ty = threadIdx.x / 16;
    for (int64_t k0 = 0; k0 < k; k0 += kDepth) {
      __syncthreads();
      for (int e = threadIdx.x; e < kTile * kDepth; e += kSimtThreads) {
        const int am = sak == 1 ? e / kDepth : e % kTile, ak = sak == 1 ? e % kDepth : e / kTile;
        as[ak][am] = m0 + am < m && k0 + ak < k ? load_f(a, (m0 + am) * sam + (k0 + ak) * sak) : 0.0f;
        const int bn = sbk == 1 ? e / kDepth : e % kTile, bk = sbk == 1 ? e % kDepth : e / kTile;
        bs[bk][bn] = n0 + bn < n && k0 + bk < k ? load_f(b, (k0 + bk) * sbk + (n0 + bn) * sbn) : 0.0f;
      }
      __syncthreads();
#pragma unroll
      for (int q = 0; q < kDepth; ++q) {
        float av[4], bv[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) av[i] = as[q][ty * 4 + i], bv[i] = bs[q][tx * 4 + i];
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int j = 0; j < 4; ++j) acc[i][j] = fmaf(av[i], bv[j], acc[i][j]);
      }
    }
  }
};

// Both products of a 64 x 64 tile, then h (dh NULL) or [dg | du] into out (M, 2 F).
template <typename T>
__global__ void __launch_bounds__(kSimtThreads)
ffn_products_kernel(const T* __restrict__ x, const T* __restrict__ wg, const T* __restrict__ wu,
                    const T* __restrict__ dh, int64_t m, int64_t k, int64_t f, int act, T* __restrict__ out) {
  __shared__ float as[kDepth][kTile + 4], bs[kDepth][kTile + 4];
  const Simt<T> simt{as, bs};
  const int64_t n0 = int64_t(blockIdx.x) * kTile, m0 = int64_t(blockIdx.y) * kTile;
  float g[4][4] = {}, u[4][4] = {};
  simt.run(x, k, 1, wg, f, 1, m0, m, n0, f, k, g);
  simt.run(x, k, 1, wu, f, 1, m0, m, n0, f, k, u);
  const int tx = threadIdx.x % 16, ty = threadIdx.x / 16;
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int64_t r = m0 + ty * 4 + i, c = n0 + tx * 4 + j;
      if (r >= m || c >= f) continue;
      float y, slope;
      activate(act, g[i][j], &y, &slope);
      if (!dh) {
        store_f(out, r * f + c, y * u[i][j]);
      } else {
        const float d = load_f(dh, r * f + c);
        store_f(out, r * 2 * f + c, d * u[i][j] * slope);
        store_f(out, r * 2 * f + f + c, d * y);
      }
    }
}

// dx = dg Wg' + du Wu'
template <typename T>
__global__ void __launch_bounds__(kSimtThreads)
ffn_dx_kernel(const T* __restrict__ dgu, const T* __restrict__ wg, const T* __restrict__ wu, int64_t m, int64_t k,
              int64_t f, T* __restrict__ dx) {
  __shared__ float as[kDepth][kTile + 4], bs[kDepth][kTile + 4];
  const Simt<T> simt{as, bs};
  const int64_t n0 = int64_t(blockIdx.x) * kTile, m0 = int64_t(blockIdx.y) * kTile;
  float acc[4][4] = {};
  simt.run(dgu, 2 * f, 1, wg, 1, f, m0, m, n0, k, f, acc);
  simt.run(dgu + f, 2 * f, 1, wu, 1, f, m0, m, n0, k, f, acc);
  const int tx = threadIdx.x % 16, ty = threadIdx.x / 16;
  for (int i = 0; i < 4; ++i)
    for (int j = 0; j < 4; ++j)
      if (m0 + ty * 4 + i < m && n0 + tx * 4 + j < k) store_f(dx, (m0 + ty * 4 + i) * k + n0 + tx * 4 + j, acc[i][j]);
}

// dW = x' [dg | du], grid.z choosing the half
template <typename T>
__global__ void __launch_bounds__(kSimtThreads)
ffn_dw_kernel(const T* __restrict__ x, const T* __restrict__ dgu, int64_t m, int64_t k, int64_t f,
              T* __restrict__ dwg, T* __restrict__ dwu) {
  __shared__ float as[kDepth][kTile + 4], bs[kDepth][kTile + 4];
  const Simt<T> simt{as, bs};
  const int64_t n0 = int64_t(blockIdx.x) * kTile, m0 = int64_t(blockIdx.y) * kTile;
  float acc[4][4] = {};
  simt.run(x, 1, k, dgu + blockIdx.z * f, 2 * f, 1, m0, k, n0, f, m, acc);
  T* dw = blockIdx.z ? dwu : dwg;
  const int tx = threadIdx.x % 16, ty = threadIdx.x / 16;
  for (int i = 0; i < 4; ++i)
    for (int j = 0; j < 4; ++j)
      if (m0 + ty * 4 + i < k && n0 + tx * 4 + j < f) store_f(dw, (m0 + ty * 4 + i) * f + n0 + tx * 4 + j, acc[i][j]);
}

constexpr int64_t kMaxExtent = int64_t(1) << 31;

int check_ffn(int dtype, int act, int64_t m, int64_t k, int64_t f) {
  if (dtype != RLENV_F32 && dtype != RLENV_BF16) return RLENV_EINVAL;
  if (act != kSilu && act != kGelu) return RLENV_EINVAL;
  if (m < 0 || k < 0 || f < 0 || m >= kMaxExtent || k >= kMaxExtent || f >= kMaxExtent / 2) return RLENV_EINVAL;
  return RLENV_OK;
}

unsigned tiles(int64_t n) { return unsigned((n + kTile - 1) / kTile); }

template <typename T>
int ffn_forward(const void* x, const void* wg, const void* wu, int64_t m, int64_t k, int64_t f, int act, void* out,
                cudaStream_t s) {
  ffn_products_kernel<T><<<dim3(tiles(f), tiles(m)), kSimtThreads, 0, s>>>(
      static_cast<const T*>(x), static_cast<const T*>(wg), static_cast<const T*>(wu), nullptr, m, k, f, act,
      static_cast<T*>(out));
  return launch_status();
}

template <typename T>
int ffn_backward(const void* dh, const void* x, const void* wg, const void* wu, int64_t m, int64_t k, int64_t f,
                 int act, void* dx, void* dwg, void* dwu, void* scratch, cudaStream_t s) {
  const T *X = static_cast<const T*>(x), *G = static_cast<const T*>(wg), *U = static_cast<const T*>(wu);
  T* dgu = static_cast<T*>(scratch);
  ffn_products_kernel<T><<<dim3(tiles(f), tiles(m)), kSimtThreads, 0, s>>>(X, G, U, static_cast<const T*>(dh), m, k, f,
                                                                           act, dgu);
  if (const int rc = launch_status()) return rc;
  ffn_dx_kernel<T><<<dim3(tiles(k), tiles(m)), kSimtThreads, 0, s>>>(dgu, G, U, m, k, f, static_cast<T*>(dx));
  if (const int rc = launch_status()) return rc;
  ffn_dw_kernel<T><<<dim3(tiles(f), tiles(k), 2), kSimtThreads, 0, s>>>(X, dgu, m, k, f, static_cast<T*>(dwg),
                                                                        static_cast<T*>(dwu));
  return launch_status();
}

}  // namespace
}  // namespace rlenv

extern "C" {

int64_t rlenv_gated_ffn_scratch_bytes(int dtype, int64_t m, int64_t k, int64_t f, int backward) {
  using namespace rlenv;
  if (check_ffn(dtype, 0, m, k, f) != RLENV_OK) return -1;
  return backward ? 2 * m * f * (dtype == RLENV_F32 ? 4 : 2) : 0;
}

int rlenv_gated_ffn_forward(int dtype, int activation, int64_t m, int64_t k, int64_t f, const void* x,
                            const void* w_gate, const void* w_up, void* out, void* scratch, int64_t scratch_bytes,
                            void* stream) {
  using namespace rlenv;
  if (const int rc = check_ffn(dtype, activation, m, k, f)) return rc;
  if (m == 0 || f == 0) return RLENV_OK;
  if (!out || (k > 0 && (!x || !w_gate || !w_up))) return RLENV_EINVAL;
  (void)scratch;
  (void)scratch_bytes;
  return dtype == RLENV_F32 ? ffn_forward<float>(x, w_gate, w_up, m, k, f, activation, out, as_stream(stream))
                            : ffn_forward<__nv_bfloat16>(x, w_gate, w_up, m, k, f, activation, out, as_stream(stream));
}

int rlenv_gated_ffn_backward(int dtype, int activation, int64_t m, int64_t k, int64_t f, const void* grad_out,
                             const void* x, const void* w_gate, const void* w_up, void* grad_x, void* grad_w_gate,
                             void* grad_w_up, void* scratch, int64_t scratch_bytes, void* stream) {
  using namespace rlenv;
  if (const int rc = check_ffn(dtype, activation, m, k, f)) return rc;
  if (m == 0 || k == 0 || f == 0) return RLENV_EINVAL;
  if (!grad_out || !x || !w_gate || !w_up || !grad_x || !grad_w_gate || !grad_w_up) return RLENV_EINVAL;
  if (!scratch_holds(scratch, scratch_bytes, rlenv_gated_ffn_scratch_bytes(dtype, m, k, f, 1))) return RLENV_EINVAL;
  return dtype == RLENV_F32
             ? ffn_backward<float>(grad_out, x, w_gate, w_up, m, k, f, activation, grad_x, grad_w_gate, grad_w_up,
                                   scratch, as_stream(stream))
             : ffn_backward<__nv_bfloat16>(grad_out, x, w_gate, w_up, m, k, f, activation, grad_x, grad_w_gate,
                                           grad_w_up, scratch, as_stream(stream));
}

}  // extern "C"
