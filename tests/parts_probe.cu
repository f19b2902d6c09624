// Test helper: the 8-bit products' joining of parts, on buffers of its caller's. Built by tests/test_lost_parts.py.
#include "int8_linear.cu"

// parts: (splits, m, f) sums; out: (m, f) float32, or bfloat16.
extern "C" int parts_probe(int floats, int splits, long long m, long long f, const int* parts, const float* a_scale,
                           const float* w_scale, void* out) {
  const unsigned blocks = unsigned((m * f + 255) / 256);
  if (floats)
    rlenv::add_parts_kernel<float><<<blocks, 256>>>(parts, splits, m, f, a_scale, w_scale, static_cast<float*>(out));
  else
    rlenv::add_parts_kernel<__nv_bfloat16><<<blocks, 256>>>(parts, splits, m, f, a_scale, w_scale,
                                                            static_cast<__nv_bfloat16*>(out));
  return int(cudaDeviceSynchronize());
}
extern "C" int parts_probe_lost() { return rlenv::kLost; }
