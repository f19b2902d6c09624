// Test helper: the bounded wait of csrc/blackwell.cuh. Built by tests/test_bounded_waits.py.
#include "blackwell.cuh"

namespace {
// One warp and a barrier. Nothing arrives: the first wait runs out after `limit` nanoseconds and sets the flag, the
// second gives up at the flag, however long it may wait. Then the flag is cleared and the phase ended: the third
// finds it over. out: the three answers, the flag after the first, and the nanoseconds that the first two took.
__global__ void wait_probe_kernel(unsigned long long limit, long long* out) {
  __shared__ __align__(8) uint64_t bar;
  __shared__ int dead;
  const uint32_t at = rlenv::bw::shared_at(&bar);
  if (threadIdx.x == 0) {
    rlenv::bw::barrier_init(at, 1);
    dead = 0;
  }
  __syncwarp();
  const uint64_t t0 = rlenv::bw::nanoseconds();
  const bool first = rlenv::bw::barrier_wait_warp(at, 0, &dead, limit);
  const uint64_t t1 = rlenv::bw::nanoseconds();
  __syncwarp();
  const int flag = *static_cast<volatile int*>(&dead);
  const bool second = rlenv::bw::barrier_wait_warp(at, 0, &dead, 1000 * limit);
  const uint64_t t2 = rlenv::bw::nanoseconds();
  __syncwarp();
  if (threadIdx.x == 0) {
    dead = 0;
    rlenv::bw::barrier_arrive(rlenv::bw::in_block(at, rlenv::bw::cluster_rank()));
  }
  __syncwarp();
  const bool third = rlenv::bw::barrier_wait_warp(at, 0, &dead, limit);
  if (threadIdx.x == 0 && flag) rlenv::bw::note_given_up();
  long long* const mine = out + 6 * threadIdx.x;
  mine[0] = first, mine[1] = second, mine[2] = third, mine[3] = flag, mine[4] = t1 - t0, mine[5] = t2 - t1;
}
}  // namespace

extern "C" int wait_probe(unsigned long long limit, long long* out) {  // out: 32 x 6
  wait_probe_kernel<<<1, 32>>>(limit, out);
  return int(cudaDeviceSynchronize());
}

extern "C" int wait_probe_status(unsigned int* count, int clear) { return rlenv::bw::read_given_up(count, clear); }

// On the host: the first of n looks at the clock, from `start` on, at which a wait of `limit` is over, or -1.
extern "C" int patience_probe(unsigned long long limit, unsigned long long start, const unsigned long long* looks, int n) {
  rlenv::bw::Patience patience(limit, start);
  for (int i = 0; i < n; ++i)
    if (patience.over(looks[i])) return i;
  return -1;
}
