// Decayed linear attention (attention.cuh): over trajectories, forward and backward, and
// one token at a time for policies that act.
#include "attention.cuh"

namespace rlenv {
namespace {

using attn::Problem;
using attn::Scan;
using attn::Strides;

constexpr int kScanThreads = 128;

// Block (seq * column tiles + tile, scan): one head of one environment from its first token to its last.
template <typename T, int D>
__global__ void __launch_bounds__(kScanThreads) scan_kernel(const __grid_constant__ Problem p) {
  constexpr int DB = D < 64 ? D : 64;
  extern __shared__ float buf[];
  const Scan& s = p.scan[blockIdx.y];
  constexpr int kTiles = D / DB;
  const int64_t seq = blockIdx.x / kTiles;
  const int col = int(blockIdx.x % kTiles) * DB;
  const int64_t n = seq / p.h, h = seq % p.h;
  attn::scan_tokens<T, D, DB, kScanThreads, true>(
      s, p, n, h, col, 0, p.t, s.carry_in ? s.carry_in + seq * D * D : nullptr, s.turned, s.in_mul, buf,
      s.carry_out ? s.carry_out + seq * D * D : nullptr, s.turned, s.out_mul);
}

template <typename T, int D>
int launch_scan(const Problem& p, cudaStream_t stream) {
  constexpr int DB = D < 64 ? D : 64;
  const int smem = int(sizeof(float)) * (D * DB + 2 * D + DB + kScanThreads);
  const dim3 grid(unsigned(p.n * p.h * (D / DB)), unsigned(p.scans));
  scan_kernel<T, D><<<grid, kScanThreads, smem, stream>>>(p);
  return launch_status();
}

// One token: S <- keep g S + k' v in place, o = scale q S. A block is one head of one environment;
// the state streams through registers once, so the kernel is bound by reading and writing it
// (8 D^2 bytes). Thread t holds four columns of every (kStepThreads * 4 / D)-th row.
constexpr int kStepThreads = 128;

template <typename T, int D>
__global__ void __launch_bounds__(kStepThreads)
step_kernel(const T* __restrict__ q, const T* __restrict__ k, const T* __restrict__ v, Strides qs, Strides ks,
            Strides vs, const float* __restrict__ decay, const uint8_t* __restrict__ resets, float scale, int64_t heads,
            float* __restrict__ state, T* __restrict__ out) {
  constexpr int kQuads = D / 4;                     // threads across a row
  constexpr int kThreads = D * D / 4 < kStepThreads ? D * D / 4 : kStepThreads;
  constexpr int kRows = kThreads / kQuads;          // rows in flight
  constexpr int kPer = D / kRows;                   // rows a thread holds
  __shared__ float part[kRows][D];
  const int64_t seq = blockIdx.x, n = seq / heads, h = seq % heads;
  const int c = (threadIdx.x % kQuads) * 4, r0 = threadIdx.x / kQuads;
  float4* S = reinterpret_cast<float4*>(state + seq * D * D);
  if (threadIdx.x < kThreads) {
    float4 z[kPer];
#pragma unroll
    for (int i = 0; i < kPer; ++i) z[i] = S[(r0 + i * kRows) * kQuads + c / 4];
    const float g = __ldg(decay + h);
    const bool reset = resets && __ldg(resets + n);
    const T* Q = q + n * qs.n + h * qs.h;
    const T* K = k + n * ks.n + h * ks.h;
    const T* V = v + n * vs.n + h * vs.h + c;
    const float v0 = attn::to_float(V[0]), v1 = attn::to_float(V[1]), v2 = attn::to_float(V[2]),
                v3 = attn::to_float(V[3]);
    float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int r = r0 + i * kRows;
      const float kr = attn::to_float(K[r]), qr = attn::to_float(Q[r]);
      float4 w = z[i];
      w.x = fmaf(kr, v0, reset ? 0.0f : g * w.x);
      w.y = fmaf(kr, v1, reset ? 0.0f : g * w.y);
      w.z = fmaf(kr, v2, reset ? 0.0f : g * w.z);
      w.w = fmaf(kr, v3, reset ? 0.0f : g * w.w);
      o.x = fmaf(qr, w.x, o.x);
      o.y = fmaf(qr, w.y, o.y);
      o.z = fmaf(qr, w.z, o.z);
      o.w = fmaf(qr, w.w, o.w);
      S[r * kQuads + c / 4] = w;
    }
    *reinterpret_cast<float4*>(&part[r0][c]) = o;
  }
  __syncthreads();
  for (int j = threadIdx.x; j < D; j += kStepThreads) {
    float sum = 0.0f;
#pragma unroll
    for (int i = 0; i < kRows; ++i) sum += part[i][j];
    out[seq * D + j] = attn::from_float<T>(scale * sum);
  }
}

bool width_built(int d) { return d == 16 || d == 32 || d == 64 || d == 128; }

// Calls fn<T, D>() for the type and width.
template <typename F>
int dispatch(int dtype, int d, F&& fn) {
  if (dtype == RLENV_F32) {
    switch (d) {
      case 16: return fn.template operator()<float, 16>();
      case 32: return fn.template operator()<float, 32>();
      case 64: return fn.template operator()<float, 64>();
      case 128: return fn.template operator()<float, 128>();
    }
  } else {
    switch (d) {
      case 16: return fn.template operator()<__nv_bfloat16, 16>();
      case 32: return fn.template operator()<__nv_bfloat16, 32>();
      case 64: return fn.template operator()<__nv_bfloat16, 64>();
      case 128: return fn.template operator()<__nv_bfloat16, 128>();
    }
  }
  return RLENV_EUNSUPPORTED;
}

// Rows are read as 16-byte pieces: a base and strides off that boundary are rejected.
bool aligned_rows(const void* p, const int64_t* st, int dtype, int axes) {
  const uint64_t size = dtype == RLENV_F32 ? 4 : 2;
  if (reinterpret_cast<uintptr_t>(p) % 16) return false;
  for (int i = 0; i < axes; ++i)
    if (uint64_t(st[i]) * size % 16) return false;
  return true;
}

struct Runner {
  const Problem& p;
  cudaStream_t stream;
  template <typename T, int D>
  int operator()() const { return launch_scan<T, D>(p, stream); }
};

constexpr int64_t kMaxBlocks = 0x7fffffff;

int check_sizes(int dtype, int d, int64_t t, int64_t n, int64_t h, float scale) {
  if (dtype != RLENV_F32 && dtype != RLENV_BF16) return RLENV_EINVAL;
  if (t < 0 || n < 0 || h < 0 || !(scale != 0.0f) || scale - scale != 0.0f) return RLENV_EINVAL;
  if (!width_built(d)) return RLENV_EUNSUPPORTED;
  if (n > 0 && h > kMaxBlocks / 2 / n) return RLENV_EINVAL;
  return RLENV_OK;
}

}  // namespace
}  // namespace rlenv

extern "C" {

int64_t rlenv_linear_attention_scratch_bytes(int dtype, int d, int64_t t, int64_t n, int64_t h, int backward) {
  using namespace rlenv;
  (void)backward;
  return check_sizes(dtype, d, t, n, h, 1.0f) == RLENV_OK ? 0 : -1;
}

int rlenv_linear_attention_forward(int dtype, int d, int64_t t, int64_t n, int64_t h, const void* q, const void* k,
                                   const void* v, const int64_t* strides, const float* decay, const uint8_t* resets,
                                   float scale, const float* state_in, void* out, float* state_out, void* scratch,
                                   int64_t scratch_bytes, void* stream) {
  using namespace rlenv;
  if (const int rc = check_sizes(dtype, d, t, n, h, scale)) return rc;
  if (n == 0 || h == 0) return RLENV_OK;
  if (t > 0 && (!q || !k || !v || !strides || !out)) return RLENV_EINVAL;
  if (!decay || !state_out || state_in == state_out) return RLENV_EINVAL;
  static const int64_t kNone[9] = {};
  const int64_t* st = t > 0 ? strides : kNone;
  if (!aligned_rows(q, st, dtype, 3) || !aligned_rows(k, st + 3, dtype, 3) || !aligned_rows(v, st + 6, dtype, 3))
    return RLENV_EINVAL;
  (void)scratch;
  (void)scratch_bytes;
  Problem p{};
  p.t = t, p.n = n, p.h = h, p.decay = decay, p.resets = resets, p.scale = scale, p.scans = 1;
  p.scan[0] = Scan{q, k, v, {st[0], st[1], st[2]}, {st[3], st[4], st[5]}, {st[6], st[7], st[8]},
                   out, state_in, state_out, 1.0f, 1.0f, 0, 0};
  return dispatch(dtype, d, Runner{p, as_stream(stream)});
}

int rlenv_linear_attention_backward(int dtype, int d, int64_t t, int64_t n, int64_t h, const void* grad_out,
                                    const void* q, const void* k, const void* v, const int64_t* strides,
                                    const float* decay, const uint8_t* resets, float scale, const float* state_in,
                                    const float* grad_state_out, void* grad_q, void* grad_k, void* grad_v,
                                    float* grad_state_in, void* scratch, int64_t scratch_bytes, void* stream) {
  using namespace rlenv;
  if (const int rc = check_sizes(dtype, d, t, n, h, scale)) return rc;
  if (n == 0 || h == 0) return RLENV_OK;
  if (t > 0 && (!grad_out || !q || !k || !v || !strides || !grad_q || !grad_k || !grad_v)) return RLENV_EINVAL;
  if (!decay || (grad_state_in && grad_state_in == grad_state_out)) return RLENV_EINVAL;
  static const int64_t kNone[12] = {};
  const int64_t* st = t > 0 ? strides : kNone;
  if (!aligned_rows(grad_out, st, dtype, 3) || !aligned_rows(q, st + 3, dtype, 3) ||
      !aligned_rows(k, st + 6, dtype, 3) || !aligned_rows(v, st + 9, dtype, 3))
    return RLENV_EINVAL;
  (void)scratch;
  (void)scratch_bytes;
  const Strides ds{st[0], st[1], st[2]}, qs{st[3], st[4], st[5]}, ks{st[6], st[7], st[8]}, vs{st[9], st[10], st[11]};
  Problem p{};
  p.t = t, p.n = n, p.h = h, p.decay = decay, p.resets = resets, p.scale = scale, p.scans = 3;
  // The reverse scans carry R / scale, so that the common factor stays outside.
  const float inv = 1.0f / scale;
  p.scan[0] = Scan{grad_out, v, k, ds, vs, ks, grad_q, state_in, nullptr, 1.0f, 1.0f, 1, 0};
  p.scan[1] = Scan{v, grad_out, q, vs, ds, qs, grad_k, grad_state_out, nullptr, inv, scale, 1, 1};
  p.scan[2] = Scan{k, q, grad_out, ks, qs, ds, grad_v, grad_state_out, grad_state_in, inv, scale, 0, 1};
  return dispatch(dtype, d, Runner{p, as_stream(stream)});
}

}  // extern "C"

namespace rlenv {
namespace {
struct StepRunner {
  const void *q, *k, *v;
  Strides qs, ks, vs;
  const float* decay;
  const uint8_t* resets;
  float scale;
  int64_t n, h;
  float* state;
  void* out;
  cudaStream_t stream;
  template <typename T, int D>
  int operator()() const {
    step_kernel<T, D><<<unsigned(n * h), kStepThreads, 0, stream>>>(
        static_cast<const T*>(q), static_cast<const T*>(k), static_cast<const T*>(v), qs, ks, vs, decay, resets, scale,
        h, state, static_cast<T*>(out));
    return launch_status();
  }
};
}  // namespace
}  // namespace rlenv

extern "C" int rlenv_linear_attention_step(int dtype, int d, int64_t n, int64_t h, const void* q, const void* k,
                                           const void* v, const int64_t* strides, const float* decay,
                                           const uint8_t* resets, float scale, float* state, void* out, void* stream) {
  using namespace rlenv;
  if (const int rc = check_sizes(dtype, d, 1, n, h, scale)) return rc;
  if (n == 0 || h == 0) return RLENV_OK;
  if (!q || !k || !v || !strides || !decay || !state || !out) return RLENV_EINVAL;
  if (!aligned_rows(q, strides, dtype, 2) || !aligned_rows(k, strides + 2, dtype, 2) ||
      !aligned_rows(v, strides + 4, dtype, 2) || reinterpret_cast<uintptr_t>(state) % 16)
    return RLENV_EINVAL;
  return dispatch(dtype, d,
                  StepRunner{q, k, v, {0, strides[0], strides[1]}, {0, strides[2], strides[3]},
                             {0, strides[4], strides[5]}, decay, resets, scale, n, h, state, out, as_stream(stream)});
}
