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

// ---------------------------------------------------------------------------
// The chunked form. kChunk tokens at a time: with Z the carry at the chunk's start,
//     out = scale (w_i x_i Z + (W * (X A')) B),    Z <- g^L Z + (l * A)' B,
// W the weights w_ij (zero above the diagonal) and l_j = g^(L - f - j) the decay from token j to
// the chunk's end: four matrix products on mma.sync with float32 accumulators.
//
// Precision. A matrix operand is a sum of 16-bit planes. bfloat16 inputs are one plane, exactly;
// float32 inputs three (8 + 8 + 8 bits of mantissa); the weighted products and the carry, which
// are float32, two for bfloat16 outputs (their own rounding is 2^-9) and three for float32 ones;
// the decayed keys three, since the carry goes out in float32. Of the products of planes those
// below 2^-24 of the whole are left out.
constexpr int kChunk = 64;

template <typename T, int D>
struct Shape {
  static constexpr bool kFloat = sizeof(T) == 4;
  static constexpr int kIn = kFloat ? 3 : 1;            // planes of x, a, b
  static constexpr int kMid = kFloat ? 3 : 2;           // of the weighted products and the carry
  static constexpr int kKeys = 3;                       // of the decayed keys
  static constexpr int DB = D < 64 ? D : 64;            // columns of the carry that a block owns
  static constexpr int PX = D + 8, PB = DB + 8;         // row pitches: 16 bytes past a multiple of 32,
                                                        // so that eight rows' pieces fall in distinct banks
  static constexpr int kX = kChunk * PX, kB = kChunk * PB, kS = D * PB;  // a plane's elements
  // Warps: kRowWarps share the chunk's tokens, kColWarps the output's columns (float32 heads of 128, whose
  // planes leave room for one block on an SM). Narrow bfloat16 heads give a warp two tiles of 16 tokens (RT): a
  // fragment of the other operand then serves twice.
  static constexpr int kRowWarps = !kFloat && D <= 32 ? 2 : 4, kColWarps = kFloat && D == 128 ? 2 : 1;
  static constexpr int kWarps = kRowWarps * kColWarps;
  static constexpr int kThreads = 32 * kWarps;
  static constexpr int RT = 4 / kRowWarps;
  static constexpr int OC = DB / kColWarps;             // output columns a warp
  // Warps change places from chunk to chunk (500 steps of 1,024 float32 heads of 64: 351 us against 386; bfloat16 heads
  // of 32: 114 against 121), but where the arithmetic of it costs as much (bfloat16 heads of 64: 243 against 233).
  static constexpr bool kTurning = kColWarps == 1 && (kFloat ? D >= 32 : D == 32);
  // Tiles come a chunk ahead: bfloat16 ones in a second buffer (cp.async), but at 128 columns, where a second
  // block on the SM is worth more; float32 ones through registers, where they become planes.
  static constexpr int kBuffers = kFloat || D == 128 ? 1 : 2;
  static constexpr int kTiles = kIn * (2 * kX + kB);    // elements of a buffer
  static constexpr int kSmem = 2 * (kBuffers * kTiles + kMid * kS);
  // The carry's rows and columns by warp: RG groups of rows, CG of columns.
  static constexpr int MT = D / 16 > kWarps ? D / 16 / kWarps : 1;  // 16-row tiles a warp
  static constexpr int RG = D / (16 * MT);
  static constexpr int CG = kWarps / RG < DB / 16 ? kWarps / RG : DB / 16;
  static constexpr int NT = DB / CG / 8;                // 8-column tiles a warp
  // blocks that fit an SM's shared memory and registers
  static constexpr int kRoom = 227 * 1024 / (kSmem + 2048), kMost = D >= 64 ? 3 : kFloat ? (D == 32 ? 3 : 4) : D == 32 ? 6 : 8;
  static constexpr int kPerSm = kRoom < kMost ? kRoom : kMost;
};

RLENV_D uint32_t shared_address(const void* p) { return uint32_t(__cvta_generic_to_shared(p)); }

RLENV_D void load_matrices(uint32_t r[4], uint32_t at) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at) : "memory");
}
RLENV_D void load_matrices_turned(uint32_t r[4], uint32_t at) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at) : "memory");
}
RLENV_D void multiply(float c[4], const uint32_t a[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
               "{%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// c (2 NT tiles of 8 columns) += a b over all pairs of planes worth it, the small ones first, `a`'s last plane
// only where `fine`; b holds two tiles a fragment. Planes run outside of tiles, so that products which add to
// the same tile are 2 NT apart: one's latency is some four others' issue. The tensor core truncates as it
// accumulates: for float32 results (three planes of data) the pairs are summed from zero and added to c in a
// rounded addition, or the error of long sums grows to a few 1e-6. bfloat16 tokens' sums do without: their results are
// rounded at 2^-9, and the float32 state that they leave is off by up to 3.4e-6 after some thousands of tokens whose
// decay is near one, far below the tokens' own rounding.
template <int NA, int NB, int NT, bool kFloat>
RLENV_D void multiply_planes(float (*c)[4], const uint32_t (&a)[NA][4], const uint32_t (&b)[NT][NB][4], bool fine = true) {
  float s[2 * NT][4] = {};
#pragma unroll
  for (int order = 2; order >= 0; --order)
#pragma unroll
    for (int u = 0; u <= order; ++u) {
      const int q = order - u;
      if (u < NA && q < NB && (u + 1 < NA || fine)) {
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          multiply(kFloat ? s[2 * t] : c[2 * t], a[u], b[t][q][0], b[t][q][1]);
          multiply(kFloat ? s[2 * t + 1] : c[2 * t + 1], a[u], b[t][q][2], b[t][q][3]);
        }
      }
    }
  if constexpr (kFloat) {
#pragma unroll
    for (int t = 0; t < 2 * NT; ++t)
#pragma unroll
      for (int q = 0; q < 4; ++q) c[t][q] += s[t][q];
  }
}

RLENV_D uint32_t pack(float lo, float hi) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}
RLENV_D float low_half(uint32_t v) { return __uint_as_float(v << 16); }
RLENV_D float high_half(uint32_t v) { return __uint_as_float(v & 0xffff0000u); }

// A pair of float32 values as N planes of bfloat16 pairs: each the rest of the ones before it.
template <int N>
RLENV_D void split_pair(float lo, float hi, uint32_t* planes, int stride) {
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const uint32_t v = pack(lo, hi);
    planes[i * stride] = v;
    lo -= low_half(v), hi -= high_half(v);
  }
}

RLENV_D void copy_async_16(uint32_t to, const void* from, bool real) {  // zeros where not real
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(real ? 16 : 0) : "memory");
}
RLENV_D void copies_end() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int kLeft>  // all but the latest kLeft groups have landed
RLENV_D void copies_landed() { asm volatile("cp.async.wait_group %0;" ::"n"(kLeft) : "memory"); }

// A thread's share of a tile of kChunk rows and W columns: 16-byte pieces of every kRowStep-th row, at a
// fixed column. `at` follows the tokens of one chunk after the other.
template <typename T, int W, int P, int kPlane, int kThreads>
struct TileLoader {
  static constexpr int kPer = 16 / sizeof(T), kPieces = W / kPer;
  static constexpr int kRowStep = kThreads / kPieces;
  static constexpr int kCount = kChunk / kRowStep;
  static_assert(kCount >= 1, "every thread has a piece");
  const T* at;
  int64_t step;  // kRowStep tokens on
  int row, col;
  RLENV_D TileLoader(const T* base, int64_t stride, bool reverse, int64_t tokens, int64_t first) {
    row = threadIdx.x / kPieces, col = threadIdx.x % kPieces * kPer;
    const int64_t i = first + row;
    at = base + (reverse ? tokens - 1 - i : i) * stride + col;
    step = (reverse ? -stride : stride) * kRowStep;
  }
  RLENV_D bool real(int u, int64_t left) const { return row + u * kRowStep < left; }
  RLENV_D void advance() { at += step * kCount; }
  // bfloat16: straight to shared memory, zeros past `left` rows
  RLENV_D void copy(uint32_t to, int64_t left) const {
#pragma unroll
    for (int u = 0; u < kCount; ++u) {
      const bool r = real(u, left);
      copy_async_16(to + ((row + u * kRowStep) * P + col) * 2, r ? at + u * step : at - row * (step / kRowStep), r);
    }
  }
  // float32: into registers, and from there as planes
  RLENV_D void fetch(float4 (&v)[kCount], int64_t left) const {
#pragma unroll
    for (int u = 0; u < kCount; ++u)
      v[u] = real(u, left) ? __ldg(reinterpret_cast<const float4*>(at + u * step)) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  }
  RLENV_D void put(__nv_bfloat16* to, const float4 (&v)[kCount]) const {
#pragma unroll
    for (int u = 0; u < kCount; ++u) {
      uint32_t lo[3], hi[3];
      split_pair<3>(v[u].x, v[u].y, lo, 1);
      split_pair<3>(v[u].z, v[u].w, hi, 1);
#pragma unroll
      for (int q = 0; q < 3; ++q)
        *reinterpret_cast<uint2*>(to + q * kPlane + (row + u * kRowStep) * P + col) = make_uint2(lo[q], hi[q]);
    }
  }
};

}  // namespace attn
}  // namespace rlenv
