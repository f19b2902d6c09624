// Products of 8-bit integers with scales: out[i][j] = (sum over k of a[i][k] w[j][k]) a_scale[i] w_scale[j], sums exact in
// 32-bit integers, scaled in float32 and rounded once to the result's type.
#include <cuda_bf16.h>

#include "common.cuh"

namespace rlenv {
namespace {

struct Int8Product {
  int64_t m, k, f;
  const int8_t *a, *w;
  int64_t a_pitch, w_pitch;
  const float *a_scale, *w_scale;
  void* out;
};

// Bytes c .. c + 15 of a row of k, zeros past its end.
RLENV_D int4 sixteen(const int8_t* row, int64_t c, int64_t k) {
  if (c + 16 <= k) return __ldg(reinterpret_cast<const int4*>(row + c));
  int w[4] = {0, 0, 0, 0};
  for (int i = 0; c + i < k; ++i) w[i / 4] |= (int(row[c + i]) & 0xff) << 8 * (i % 4);
  return make_int4(w[0], w[1], w[2], w[3]);
}
RLENV_D int dot(int4 a, int4 b, int sum) {
  return __dp4a(a.w, b.w, __dp4a(a.z, b.z, __dp4a(a.y, b.y, __dp4a(a.x, b.x, sum))));
}
RLENV_D void put(float* to, float x) { *to = x; }
RLENV_D void put(__nv_bfloat16* to, float x) { *to = __float2bfloat16_rn(x); }

// Few rows: a warp for kChannels channels, which reads their weights once for kRows rows.
template <typename T, int kRows, int kChannels>
__global__ void __launch_bounds__(256) few_rows_kernel(const __grid_constant__ Int8Product p) {
  const int lane = threadIdx.x % 32;
  const int64_t f0 = (int64_t(blockIdx.x) * 8 + threadIdx.x / 32) * kChannels, m0 = int64_t(blockIdx.y) * kRows;
  if (f0 >= p.f) return;
  int sums[kRows][kChannels] = {};
  for (int64_t c = 16 * lane; c < p.k; c += 512) {
    int4 w[kChannels];
#pragma unroll
    for (int j = 0; j < kChannels; ++j) w[j] = f0 + j < p.f ? sixteen(p.w + (f0 + j) * p.w_pitch, c, p.k) : make_int4(0, 0, 0, 0);
#pragma unroll
    for (int i = 0; i < kRows; ++i) {
      if (m0 + i >= p.m) break;
      const int4 a = sixteen(p.a + (m0 + i) * p.a_pitch, c, p.k);
#pragma unroll
      for (int j = 0; j < kChannels; ++j) sums[i][j] = dot(a, w[j], sums[i][j]);
    }
  }
#pragma unroll
  for (int i = 0; i < kRows; ++i)
#pragma unroll
    for (int j = 0; j < kChannels; ++j) {
      const int sum = __reduce_add_sync(0xffffffffu, sums[i][j]);
      if (lane == 0 && m0 + i < p.m && f0 + j < p.f)
        put(static_cast<T*>(p.out) + (m0 + i) * p.f + f0 + j, float(sum) * p.a_scale[m0 + i] * p.w_scale[f0 + j]);
    }
}

template <typename T>
int product(const Int8Product& p, cudaStream_t s) {
  const dim3 grid(unsigned((p.f + 31) / 32), unsigned((p.m + 7) / 8));
  few_rows_kernel<T, 8, 4><<<grid, 256, 0, s>>>(p);
  return launch_status();
}

bool int8_sizes(int64_t m, int64_t k, int64_t f) {
  return m >= 0 && f >= 0 && k >= 1 && k <= 131071 && m < 65535 * 8 && f < (int64_t(1) << 31);
}
bool on_boundary(const void* p, int size) { return p && reinterpret_cast<uintptr_t>(p) % size == 0; }

}  // namespace
}  // namespace rlenv

extern "C" {

int64_t rlenv_int8_linear_scratch_bytes(int64_t m, int64_t k, int64_t f) {
  return rlenv::int8_sizes(m, k, f) ? 0 : RLENV_EINVAL;
}

int rlenv_int8_linear_forward(int dtype, int64_t m, int64_t k, int64_t f, const int8_t* a, int64_t a_pitch,
                              const float* a_scale, const int8_t* w, int64_t w_pitch, const float* w_scale, void* out,
                              void* scratch, int64_t scratch_bytes, void* stream) {
  using namespace rlenv;
  if ((dtype != RLENV_F32 && dtype != RLENV_BF16) || !int8_sizes(m, k, f) || a_pitch < k || w_pitch < k || a_pitch % 16 ||
      w_pitch % 16)
    return RLENV_EINVAL;
  if (m == 0 || f == 0) return RLENV_OK;
  if (!on_boundary(a, 16) || !on_boundary(w, 16) || !on_boundary(a_scale, 4) || !on_boundary(w_scale, 4) ||
      !on_boundary(out, dtype == RLENV_F32 ? 4 : 2) ||
      !scratch_holds(scratch, scratch_bytes, rlenv_int8_linear_scratch_bytes(m, k, f)))
    return RLENV_EINVAL;
  const Int8Product p{m, k, f, a, w, a_pitch, w_pitch, a_scale, w_scale, out};
  return dtype == RLENV_F32 ? product<float>(p, as_stream(stream)) : product<__nv_bfloat16>(p, as_stream(stream));
}

}  // extern "C"
