// Decayed linear attention over trajectories: the pieces that the kernels of
// attention.cu share.
//
// One head of one environment carries a D x D state S. A token with query q, key k and
// value v does
//     S <- keep g S + k' v,    o = scale q S,
// g in [0, 1] the head's decay and keep = 0 where the token starts an episode. The
// gradients are scans of the same kind. With R_t = scale q_t' do_t + keep_{t+1} g R_{t+1}
// (R of the last token also holds the gradient of the final state)
//     dq_t = scale do_t S_t',    dk_t = v_t R_t',    dv_t = k_t R_t,
// so that every one of the four is
//     out_i = scale (sum_{j <= i} w_ij (x_i . a_j) b_j + w_i x_i Z)
// with (x, a, b) = (q, k, v), (do, v, k), (v, do, q), (k, q, do), the last two from the
// last token to the first. `Scan` describes one. In scan order the weights are
//     w_ij = g^(i - j) where no reset lies between,  w_i = g^(i + f),  f = 1 forward,
// f = 0 in reverse, where a token is read before its decay is applied. A reset acts before
// its token is used going forward and after it in reverse.
#pragma once

#include <cuda_bf16.h>

#include "common.cuh"

namespace rlenv {
namespace attn {

struct Strides {  // elements between steps, environments and heads; the last axis is dense
  int64_t t, n, h;
};

struct Scan {
  const void *x, *a, *b;
  Strides xs, as, bs;
  void* out;              // (T, N, H, D) dense, of the inputs' type
  const float* carry_in;  // (N, H, D, D) or NULL for zero
  float* carry_out;       // or NULL
  float in_mul, out_mul;  // factors of the carry on its way in and out
  int turned;             // the carry is stored transposed (b's axis first)
  int reverse;
};

struct Problem {
  int64_t t, n, h;
  const float* decay;      // (H,)
  const uint8_t* resets;   // (T, N) or NULL
  float scale;
  int scans;
  Scan scan[3];
};

template <typename T>
RLENV_D float to_float(T x) { return float(x); }
template <>
RLENV_D float to_float<__nv_bfloat16>(__nv_bfloat16 x) { return __bfloat162float(x); }
template <typename T>
RLENV_D T from_float(float x) { return T(x); }
template <>
RLENV_D __nv_bfloat16 from_float<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }

// g^n for n >= 0 (g^0 = 1 for every g, zero and NaN too).
RLENV_D float power(float log2_g, int64_t n) { return n == 0 ? 1.0f : exp2f(float(n) * log2_g); }

// Positions [first, last) in scan order, token by token: the definition itself, which the chunked
// kernel falls back to where a value is not finite (a masked product is zero there only if nothing
// masked is infinite or NaN; here what a reset cuts off is dropped by a select). The block owns
// columns [col, col + DB) of the state, held in shared memory: thread t column t % DB, rows strided
// by the threads left. `buf` needs (D * DB + 2 * D + DB + threads) floats. state_in points at the carry
// for position `first` (NULL: zero); with WRITE_OUT unset only the state is formed.
template <typename T, int D, int DB, int kBlock, bool kWriteOut>
RLENV_D void scan_tokens(const Scan& s, const Problem& p, int64_t n, int64_t h, int col, int64_t first,
                         int64_t last, const float* carry, bool carry_turned, float carry_mul, float* buf,
                         float* state_out, bool out_turned, float out_mul) {
  float* S = buf;
  float* xv = S + D * DB;
  float* av = xv + D;
  float* bv = av + D;
  float* part = bv + DB;
  const int c = threadIdx.x % DB, r0 = threadIdx.x / DB;
  constexpr int kRows = kBlock / DB;
  const float g = __ldg(p.decay + h);
  const T* X = static_cast<const T*>(s.x) + n * s.xs.n + h * s.xs.h;
  const T* A = static_cast<const T*>(s.a) + n * s.as.n + h * s.as.h;
  const T* B = static_cast<const T*>(s.b) + n * s.bs.n + h * s.bs.h + col;
  __syncthreads();
  for (int r = r0; r < D; r += kRows)
    S[r * DB + c] = carry ? carry_mul * __ldg(carry + (carry_turned ? (col + c) * D + r : r * D + col + c)) : 0.0f;
  for (int64_t i = first; i < last; ++i) {
    const int64_t t = s.reverse ? p.t - 1 - i : i;
    const bool reset = p.resets && __ldg(p.resets + t * p.n + n);
    __syncthreads();
    for (int r = threadIdx.x; r < D; r += kBlock) {
      if (kWriteOut) xv[r] = to_float(X[t * s.xs.t + r]);
      av[r] = to_float(A[t * s.as.t + r]);
      if (r < DB) bv[r] = to_float(B[t * s.bs.t + r]);
    }
    __syncthreads();
    float acc = 0.0f;
    for (int r = r0; r < D; r += kRows) {
      float z = S[r * DB + c];
      if (!s.reverse) z = reset ? 0.0f : g * z;
      z = fmaf(av[r], bv[c], z);
      if (kWriteOut) acc = fmaf(xv[r], z, acc);
      if (s.reverse) z = reset ? 0.0f : g * z;
      S[r * DB + c] = z;
    }
    if (kWriteOut) {
      part[threadIdx.x] = acc;
      __syncthreads();
      if (threadIdx.x < DB) {
        float sum = 0.0f;
        for (int q = 0; q < kRows; ++q) sum += part[q * DB + c];
        static_cast<T*>(s.out)[((t * p.n + n) * p.h + h) * D + col + c] = from_float<T>(p.scale * sum);
      }
    }
  }
  if (state_out)
    for (int r = r0; r < D; r += kRows)
      state_out[out_turned ? (col + c) * D + r : r * D + col + c] = out_mul * S[r * DB + c];
}

}  // namespace attn
}  // namespace rlenv
