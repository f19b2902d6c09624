// The sm_100a instructions that the matrix kernels are written with: barriers in shared memory,
// tensor copies, and the tensor cores with their accumulators in tensor memory.
#pragma once

#include <cuda.h>

#include "common.cuh"

namespace rlenv {
namespace bw {

RLENV_D uint32_t shared_at(const void* p) { return uint32_t(__cvta_generic_to_shared(p)); }

// ---- barriers ---------------------------------------------------------------------------------
RLENV_D void barrier_init(uint32_t bar, uint32_t count) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count) : "memory");
}
// The same place in the shared memory of block `rank` of the cluster.
RLENV_D uint32_t in_block(uint32_t at, uint32_t rank) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(at), "r"(rank));
  return r;
}
// (Default scopes, here and in the waits: what passes between the blocks is tensor memory, ordered by
// tcgen05.fence, and shared memory, ordered by the copies' and products' own arrivals. At cluster scope
// each would carry a fence of all memory.)
RLENV_D void barrier_arrive(uint32_t cluster_bar) {
  asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(cluster_bar) : "memory");
}
RLENV_D void barrier_expect(uint32_t bar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
// Bytes that will not come count as come.
RLENV_D void barrier_strike(uint32_t bar, uint32_t bytes) {
  asm volatile("mbarrier.complete_tx.relaxed.cluster.shared::cluster.b64 [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
RLENV_D void store_in_block(uint32_t cluster_at, int x) {
  asm volatile("st.shared::cluster.b32 [%0], %1;" ::"r"(cluster_at), "r"(x) : "memory");
}
RLENV_D bool barrier_try(uint32_t bar, uint32_t parity) {
  uint32_t done;
  asm volatile(
      "{\n .reg .pred p;\n mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n selp.u32 %0, 1, 0, p;\n}"
      : "=r"(done) : "r"(bar), "r"(parity) : "memory");
  return done != 0;
}
// Waits for the phase of `parity` to end. Every wait is bounded: after kPatience nanoseconds `dead` is set,
// and from then on every wait of the block gives up at once. What counts is time between looks at the barrier, of
// each pause kLongestPause at most: while the GPU runs another process's kernels, the clock goes on and the block
// does not, nor what it waits for.
constexpr uint64_t kPatience = 2000000000, kLongestPause = 10000000;
struct Patience {
  uint64_t limit, last, waited;
  RLENV_HD Patience(uint64_t limit, uint64_t now) : limit(limit), last(now), waited(0) {}
  RLENV_HD bool over(uint64_t now) {
    const uint64_t pause = now - last;
    waited += pause < kLongestPause ? pause : kLongestPause;
    last = now;
    return waited > limit;
  }
};
RLENV_D uint64_t nanoseconds() {
  uint64_t t;
  asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t));
  return t;
}
// A whole warp waits, all of whose lanes get the same answer, and know it: copies and products take their
// operands from the warp's uniform registers, and under control flow that may diverge each operand is moved there
// anew, some 60 cycles a product. So the warps that issue them run as one, and only the instruction itself stands
// under `elect`.
RLENV_D bool barrier_wait_warp(uint32_t bar, uint32_t parity, volatile int* dead, uint64_t limit = kPatience) {
  for (int i = 0; i < 32; ++i)
    if (__all_sync(0xffffffffu, barrier_try(bar, parity))) return true;
  Patience patience(limit, nanoseconds());
  while (true) {
    if (__all_sync(0xffffffffu, barrier_try(bar, parity))) return true;
    if (__any_sync(0xffffffffu, *dead != 0)) return false;
    if (__any_sync(0xffffffffu, patience.over(nanoseconds()))) break;
  }
  *dead = 1;
  return false;
}

// Blocks that have ended with a wait that ran out, of this source file's kernels and on this device. The reader
// waits for the device: streams that do not wait for the default one hold launches too.
static __device__ unsigned int g_given_up;
RLENV_D void note_given_up() { atomicAdd(&g_given_up, 1u); }
static inline int read_given_up(unsigned int* count, bool clear) {
  const unsigned int zero = 0;
  if (cudaError_t e = cudaDeviceSynchronize()) return int(e);
  if (cudaError_t e = cudaMemcpyFromSymbol(count, g_given_up, sizeof zero)) return int(e);
  return clear ? int(cudaMemcpyToSymbol(g_given_up, &zero, sizeof zero)) : RLENV_OK;
}

RLENV_D bool elect() {  // one lane of the warp
  uint32_t r;
  asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.u32 %0, 1, 0, p;\n}" : "=r"(r));
  return r != 0;
}

// ---- tensor copies ------------------------------------------------------------------------------
// Into this block's shared memory; the bytes are counted at a barrier of either block of the pair.
RLENV_D void copy_tile(uint32_t to, const CUtensorMap* map, uint32_t cluster_bar, int x, int y, int z) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.cta_group::2 "
      "[%0], [%1, {%3, %4, %5}], [%2];" ::"r"(to),
      "l"(map), "r"(cluster_bar), "r"(x), "r"(y), "r"(z)
      : "memory");
}
RLENV_D uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
RLENV_D void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n barrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// ---- tensor memory and tensor cores ---------------------------------------------------------------
// The two blocks of a cluster work as a pair (cta_group::2): a product of 2 x 128 rows has each block's
// rows of A and half of B's columns in its own shared memory, and each block's rows of the result in its
// own tensor memory. Allocation is a matter of both blocks, products of the first block's one thread.
template <int kColumns>
RLENV_D void tmem_alloc(uint32_t slot) {  // one warp
  asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(slot), "r"(kColumns) : "memory");
  asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
}
template <int kColumns>
RLENV_D void tmem_free(uint32_t at) {  // the same warp
  asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(at), "r"(kColumns) : "memory");
}
RLENV_D void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
RLENV_D void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
// Arrives at `bar` of both blocks when the matrix products issued so far are done.
RLENV_D void commit(uint32_t bar) {
  asm volatile(
      "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(bar),
      "h"(uint16_t(3))
      : "memory");
}
// The high word of every operand's descriptor: eight rows every 1,024 bytes, 128-byte swizzle.
constexpr uint32_t kOperandHigh = 1024 >> 4 | 1u << 14 | 2u << 29;

// D (+)= A B; a and b are the operands' places (below). One thread issues a product after the other, each
// waiting for the few instructions before it, so nothing is computed here that can stand outside the loop.
RLENV_D void multiply(uint32_t d, uint32_t a, uint32_t b, uint32_t kind, bool accumulate) {
  asm volatile(
      "{\n .reg .pred p;\n .reg .b64 a, b;\n setp.ne.b32 p, %4, 0;\n mov.b64 a, {%1, %5};\n mov.b64 b, {%2, %5};\n"
      " tcgen05.mma.cta_group::2.kind::f16 [%0], a, b, %3, p;\n}" ::"r"(d),
      "r"(a), "r"(b), "r"(kind), "r"(uint32_t(accumulate)), "n"(kOperandHigh)
      : "memory");
}
// 16 columns at each of two places, of this warp's 32 lanes: lane l gets its row's columns, as bits. They are
// there after tmem_ready, which takes the registers through, so that no use of them comes before it.
RLENV_D void tmem_load16x2(uint32_t (&r)[32], uint32_t at, uint32_t and_at) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%32];\n"
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%33];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
        "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
        "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(at), "r"(and_at)
      : "memory");
}
RLENV_D void tmem_ready(uint32_t (&r)[32]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]),
                 "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]),
                 "+r"(r[16]), "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]), "+r"(r[22]), "+r"(r[23]),
                 "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]), "+r"(r[29]), "+r"(r[30]), "+r"(r[31])
               :
               : "memory");
}

// The place of a bfloat16 operand in shared memory, rows of 128 bytes swizzled by eights as the tensor
// copies write them: the low word of its descriptor, in 16-byte units, so that `bytes` further on is an
// addition of bytes / 16. K-major: a row is 64 elements of the contraction, eight rows 1,024 bytes apart from
// the next eight. MN-major: a row is 64 elements of the other axis, eight steps of the contraction 1,024 bytes
// apart from the next eight and the next 64 elements `block` bytes away.
RLENV_D uint32_t operand(uint32_t at, bool mn_major, uint32_t block) {
  return (at & 0x3ffff) >> 4 | (mn_major ? block >> 4 : 1) << 16;
}
// bfloat16 x bfloat16 -> float32, M x N.
constexpr uint32_t product_kind(int m, int n, bool a_mn, bool b_mn) {
  return 1u << 4 | 1u << 7 | 1u << 10 | uint32_t(a_mn) << 15 | uint32_t(b_mn) << 16 | uint32_t(n >> 3) << 17 |
         uint32_t(m >> 4) << 24;
}

// ---- host: tensor maps -----------------------------------------------------------------------------
using EncodeTiled = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                 const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                 CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

inline EncodeTiled encode_tiled() {  // the driver's function, looked up once
  static const EncodeTiled fn = [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult found;
    if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &p, 12000, cudaEnableDefault, &found) != cudaSuccess ||
        found != cudaDriverEntryPointSuccess)
      p = nullptr;
    return reinterpret_cast<EncodeTiled>(p);
  }();
  return fn;
}

// A (slices, rows, cols) bfloat16 array with `pitch` elements between rows, copied in boxes of 64
// columns and box_rows rows; what lies past cols or rows reads as zero. 0 or a cudaError_t.
inline int tile_map(CUtensorMap* map, const void* base, int64_t cols, int64_t rows, int64_t slices, int64_t pitch,
                    int box_rows) {
  const EncodeTiled encode = encode_tiled();
  if (!encode) return int(cudaErrorNotSupported);
  const cuuint64_t dims[3] = {cuuint64_t(cols), cuuint64_t(rows), cuuint64_t(slices)};
  const cuuint64_t strides[2] = {cuuint64_t(pitch) * 2, cuuint64_t(pitch) * 2 * cuuint64_t(rows)};
  const cuuint32_t box[3] = {64, cuuint32_t(box_rows), 1}, steps[3] = {1, 1, 1};
  const CUresult rc = encode(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void*>(base), dims, strides, box,
                             steps, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                             CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return rc == CUDA_SUCCESS ? 0 : int(cudaErrorInvalidValue);
}

}  // namespace bw
}  // namespace rlenv
