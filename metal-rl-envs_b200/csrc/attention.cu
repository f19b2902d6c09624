// Decayed linear attention (attention.cuh): over trajectories, forward and backward, and
// one token at a time for policies that act.
#include "attention.cuh"

namespace rlenv {
namespace {

using attn::Problem;
using attn::Scan;
using attn::Strides;

// A sequence (one head of one environment) or, where there are few of them, a segment of one:
// `segments` runs of `per` chunks. Split sequences take three launches: chunk_kernel<local> forms each
// segment's own carry from zero, join_kernel the carry at each segment's start, and
// chunk_kernel<whole> the outputs.
//
// Measured: bfloat16 heads of 64, 500 steps x 256 x 8, 230 us (2.6 TB/s of the tensors; the tensor pipe 45% busy,
// shared memory 61%, issue 42%: a warp's fragments come from shared memory, and what a warp waits for next is
// hidden by two other warps of its scheduler only); gradient of half as many 328 us. float32 heads of 128, 16,384
// steps x 8, 420 us, of which 101 us are the segments' own carries and 8 us the joining.
struct Split {
  int64_t segments, per;
  float* carry;    // (scans, sequences, segments, D, D): a segment's own, then the one at its start
  float* through;  // (scans, sequences, segments): the decay over a segment, -1 where a reset cuts it
};

template <typename T, int D, bool kLocal>
__global__ void __launch_bounds__(attn::Shape<T, D>::kThreads, attn::Shape<T, D>::kPerSm)
chunk_kernel(const __grid_constant__ Problem p, const __grid_constant__ Split split) {
  using namespace attn;
  using C = Shape<T, D>;
  constexpr int DB = C::DB, kTiles = D / DB;
  extern __shared__ __align__(16) unsigned char smem[];
  __shared__ float powers[kChunk + 17];  // of the decay
  __nv_bfloat16* const tiles = reinterpret_cast<__nv_bfloat16*>(smem);
  __nv_bfloat16* const S = tiles + C::kBuffers * C::kTiles;
  constexpr int kAAt = C::kIn * C::kX, kBAt = 2 * C::kIn * C::kX;  // x, a and b in a buffer

  uint32_t id = blockIdx.x;  // the counts that make it up are below 2^31 as it is
  const int col = int(id % kTiles) * DB;
  id /= kTiles;
  const uint32_t scan = p.scans == 1 ? 0 : id % p.scans;
  const Scan& s = p.scan[scan];
  id /= p.scans;
  const uint32_t segments = uint32_t(split.segments), seq = segments == 1 ? id : id / segments;
  const int64_t segment = id - seq * segments;
  const int64_t n = seq / uint32_t(p.h), h = seq % uint32_t(p.h);
  const int64_t slot = (scan * p.n * p.h + seq) * segments + segment;
  const int64_t first = segment * split.per * kChunk;
  const int64_t last = first + split.per * kChunk < p.t ? first + split.per * kChunk : p.t;
  const bool whole = segments == 1;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  // This warp's first 16 tokens and output columns. Later tokens have more before them, and a scheduler has the same
  // warps of every block: the warps of the other columns stand the other way round (float32 heads of 128, 16,384
  // tokens: 311 us against 356), and those of Shape::kTurning change places from chunk to chunk.
  int rb = warp % C::kRowWarps * C::RT;
  if (warp >= C::kRowWarps) rb = (C::kRowWarps - 1) * C::RT - rb;
  const int oc = warp / C::kRowWarps * C::OC;
  const int gr = lane >> 2, gc = (lane & 3) * 2;      // a fragment's row and column
  const float log2_g = log2f(__ldg(p.decay + h));
  const int f = s.reverse ? 0 : 1;
  for (int j = threadIdx.x; j < kChunk + 17; j += C::kThreads) powers[j] = power(log2_g, j);

  // The carry, float32 in registers: rows srow + 16 m + (gr, gr + 8), columns scol + 8 t + (gc, gc + 1).
  const int rg = warp % C::RG, cg = warp / C::RG;
  const bool holds = cg < C::CG;
  const int srow = rg * 16 * C::MT, scol = cg * 8 * C::NT;
  const bool fine = kLocal || C::kFloat || s.carry_out;  // a carry that goes out in float32 takes all planes
  float z[C::MT][C::NT][4];
  const float* start = kLocal ? nullptr : whole ? s.carry_in : split.carry + slot * D * D;
  if (!kLocal && whole && start) start += int64_t(seq) * D * D;
  const bool turned = whole && s.turned;
  const float start_mul = whole ? s.in_mul : 1.0f;
#pragma unroll
  for (int m = 0; m < C::MT; ++m)
#pragma unroll
    for (int t = 0; t < C::NT; ++t)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int r = srow + 16 * m + gr + (q & 2) * 4, c = col + scol + 8 * t + gc + (q & 1);
        z[m][t][q] = start && holds ? start_mul * __ldg(start + (turned ? c * D + r : r * D + c)) : 0.0f;
      }

  using LoadX = TileLoader<T, D, C::PX, C::kX, C::kThreads>;
  using LoadB = TileLoader<T, DB, C::PB, C::kB, C::kThreads>;
  LoadX load_x(static_cast<const T*>(s.x) + n * s.xs.n + h * s.xs.h, s.xs.t, s.reverse, p.t, first);
  LoadX load_a(static_cast<const T*>(s.a) + n * s.as.n + h * s.as.h, s.as.t, s.reverse, p.t, first);
  LoadB load_b(static_cast<const T*>(s.b) + n * s.bs.n + h * s.bs.h + col, s.bs.t, s.reverse, p.t, first);
  float4 vx[C::kFloat && !kLocal ? LoadX::kCount : 1], va[C::kFloat ? LoadX::kCount : 1], vb[C::kFloat ? LoadB::kCount : 1];
  // the next chunk's tiles set out, from chunk `i` into buffer `to`
  const auto set_out = [&](int64_t i, __nv_bfloat16* to) {
    if constexpr (C::kFloat) {
      if constexpr (!kLocal) load_x.fetch(vx, last - i);
      load_a.fetch(va, last - i);
      load_b.fetch(vb, last - i);
    } else {
      if constexpr (!kLocal) load_x.copy(shared_address(to), last - i);
      load_a.copy(shared_address(to + kAAt), last - i);
      load_b.copy(shared_address(to + kBAt), last - i);
      copies_end();
    }
    load_x.advance(), load_a.advance(), load_b.advance();
  };
  // a lane's two resets of a chunk, as bytes
  const int64_t reset_step = s.reverse ? -p.n : p.n;
  const uint8_t* reset_at = p.resets + (s.reverse ? p.t - 1 - (first + lane) : first + lane) * p.n + n;
  int reset0 = 0, reset1 = 0;
  const auto read_resets = [&](int64_t i) {
    reset0 = i + lane < last ? __ldg(reset_at) : 0;
    reset1 = i + 32 + lane < last ? __ldg(reset_at + 32 * reset_step) : 0;
    reset_at += kChunk * reset_step;
  };
  // results leave as 16-byte pieces: lane l the piece l % kPieces of row l / kPieces of the warp's
  constexpr int kPer = 16 / sizeof(T), kPieces = C::OC / kPer, kRowsOut = 32 / kPieces;
  const int64_t token_step = p.n * p.h * D, out_step = s.reverse ? -token_step : token_step;
  T* out_at;
  {
    const int64_t i = first + (C::kTurning ? 0 : 16 * rb) + lane / kPieces;
    out_at = static_cast<T*>(s.out) + (s.reverse ? p.t - 1 - i : i) * token_step + int64_t(seq) * D + col + oc + lane % kPieces * kPer;
  }
  if (p.resets && first < last) read_resets(first);
  constexpr bool kAhead = C::kFloat || C::kBuffers == 2;  // tiles set out a chunk ahead
  if (kAhead && first < last) set_out(first, tiles);
  __syncthreads();  // the powers are there

  // The weights, `scale` among them, between 16 tokens and 16 others: on the diagonal, and one block to its
  // left; and from the carry to this warp's tokens.
  float near[8], next[8], row_decay[C::RT][2];
  const auto decay_rows = [&] {
#pragma unroll
    for (int r = 0; r < C::RT; ++r)
#pragma unroll
      for (int half = 0; half < 2; ++half) row_decay[r][half] = p.scale * powers[16 * (rb + r) + gr + 8 * half + f];
  };
  if constexpr (!kLocal) {
#pragma unroll
    for (int q = 0; q < 8; ++q) {
      const int apart = gr + (q & 2) * 4 - (gc + (q & 1) + (q & 4) * 2);
      near[q] = apart >= 0 ? p.scale * powers[apart] : 0.0f;
      next[q] = p.scale * powers[16 + apart];
    }
    decay_rows();
  }
  const float block_decay = powers[16];

  float bad = 0.0f;      // NaN once any value is not finite
  bool cut = false;      // a reset anywhere in the segment
  int buffer = 0;
  for (int64_t i0 = first; i0 < last; i0 += kChunk) {
    const int len = int(last - i0 < kChunk ? last - i0 : kChunk);
    // Blocks of 16 tokens that hold any; wide heads, whose time goes with the carry, work on all four and keep
    // their loops straight.
    const int live = D <= 32 || (C::kFloat && D == 64) ? (len + 15) / 16 : kChunk / 16;
    __nv_bfloat16* const X = tiles + buffer * C::kTiles;
    __nv_bfloat16* const A = X + kAAt;
    __nv_bfloat16* const B = X + kBAt;
    if (C::kBuffers == 2) buffer ^= 1;
    if (!kAhead) set_out(i0, tiles);
    uint64_t resets = 0;
    if (p.resets) {
      resets = uint64_t(__ballot_sync(0xffffffffu, reset1 != 0)) << 32 | __ballot_sync(0xffffffffu, reset0 != 0);
      cut = cut || resets != 0;
    }
    // The first position that position i (or, for i = 63, the chunk's end) is linked to; `none`: also the carry.
    const auto linked_from = [&](uint64_t before, bool* none) -> int {
      const uint64_t m = resets & before;
      *none = m == 0;
      return m ? 64 - f - __clzll(m) : 0;
    };
    if constexpr (!kLocal) {
      // the carry at the chunk's start as planes
      if (holds) {
#pragma unroll
        for (int m = 0; m < C::MT; ++m)
#pragma unroll
          for (int t = 0; t < C::NT; ++t)
#pragma unroll
            for (int half = 0; half < 2; ++half) {
              uint32_t v[C::kMid];
              split_pair<C::kMid>(z[m][t][2 * half], z[m][t][2 * half + 1], v, 1);
#pragma unroll
              for (int q = 0; q < C::kMid; ++q)
                *reinterpret_cast<uint32_t*>(S + q * C::kS + (srow + 16 * m + gr + 8 * half) * C::PB + scol + 8 * t +
                                             gc) = v[q];
            }
      }
    }
    if constexpr (C::kFloat) {
      if constexpr (!kLocal) load_x.put(X, vx);
      load_a.put(A, va);
      load_b.put(B, vb);
    } else {
      copies_landed<0>();
    }
    __syncthreads();
    const int64_t next_chunk = i0 + kChunk;
    if (next_chunk < last) {
      if (kAhead) set_out(next_chunk, tiles + buffer * C::kTiles);
      if (p.resets) read_resets(next_chunk);
    }
    __syncwarp();  // lanes part where a tile's rows end; the matrix instructions are the whole warp's

    if (!kLocal && rb < live) {
      float o[C::RT][C::OC / 8][4];
#pragma unroll
      for (int r = 0; r < C::RT; ++r)
#pragma unroll
        for (int t = 0; t < C::OC / 8; ++t)
#pragma unroll
          for (int q = 0; q < 4; ++q) o[r][t][q] = 0.0f;
      const uint32_t xa = shared_address(X + (16 * rb + (lane & 15)) * C::PX + (lane >> 4) * 8);
      const uint32_t sa = shared_address(S + (lane & 15) * C::PB + (lane >> 4) * 8 + oc);
      constexpr int kGroup = C::OC >= 32 ? 2 : 1;  // pairs of tiles whose products run side by side
      const auto load_x_tiles = [&](uint32_t (&x)[C::RT][C::kIn][4], int k) {
#pragma unroll
        for (int r = 0; r < C::RT; ++r)
#pragma unroll
          for (int q = 0; q < C::kIn; ++q) load_matrices(x[r][q], xa + 2 * (q * C::kX + 16 * r * C::PX + 16 * k));
      };
      // Tokens of bfloat16 heads of 64 stay in registers for all of their products (the rollouts 230 us against 233;
      // wider heads have no registers left, narrower ones no use for it).
      constexpr int kKept = !C::kFloat && D == 64 ? D / 16 : 0;
      uint32_t kept[kKept ? kKept : 1][C::RT][C::kIn][4];
#pragma unroll
      for (int k = 0; k < kKept; ++k) load_x_tiles(kept[k], k);
      // x Z
#pragma unroll
      for (int k = 0; k < D / 16; ++k) {
        uint32_t fresh[C::RT][C::kIn][4];
        if (!kKept) load_x_tiles(fresh, k);
        const auto& x = kKept ? kept[kKept ? k : 0] : fresh;
#pragma unroll
        for (int t = 0; t < C::OC / 16; t += kGroup) {
          uint32_t v[kGroup][C::kMid][4];
#pragma unroll
          for (int i = 0; i < kGroup; ++i)
#pragma unroll
            for (int q = 0; q < C::kMid; ++q)
              load_matrices_turned(v[i][q], sa + 2 * (q * C::kS + 16 * k * C::PB + 16 * (t + i)));
#pragma unroll
          for (int r = 0; r < C::RT; ++r)
            multiply_planes<C::kIn, C::kMid, kGroup, C::kFloat>(&o[r][2 * t], x[r], v);
        }
      }
      int from[C::RT][2] = {};
#pragma unroll
      for (int r = 0; r < C::RT; ++r)
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          bool carry = true;
          if (resets) from[r][half] = linked_from((uint64_t(f + 1) << (16 * (rb + r) + gr + 8 * half)) - 1, &carry);
          const float keep = row_decay[r][half];
#pragma unroll
          for (int t = 0; t < C::OC / 8; ++t) {
            o[r][t][2 * half] = carry ? keep * o[r][t][2 * half] : 0.0f;
            o[r][t][2 * half + 1] = carry ? keep * o[r][t][2 * half + 1] : 0.0f;
          }
        }
      // (W * x a') b, 16 tokens at a time from the diagonal to the left
      const uint32_t aa = shared_address(A + ((lane & 7) + (lane >> 4) * 8) * C::PX + ((lane >> 3) & 1) * 8);
      const uint32_t ba = shared_address(B + (lane & 15) * C::PB + (lane >> 4) * 8 + oc);
      float far[C::RT];
#pragma unroll
      for (int r = 0; r < C::RT; ++r) far[r] = 1.0f;
      for (int jb = min(rb + C::RT, live) - 1; jb >= 0; --jb) {
        float w[C::RT][2][4] = {}, w_odd[C::RT][2][4] = {};  // even and odd steps of the sum side by side
#pragma unroll
        for (int k = 0; k < D / 16; ++k) {
          uint32_t fresh[C::RT][C::kIn][4], v[1][C::kIn][4];
          if (!kKept) load_x_tiles(fresh, k);
          const auto& x = kKept ? kept[kKept ? k : 0] : fresh;
#pragma unroll
          for (int q = 0; q < C::kIn; ++q) load_matrices(v[0][q], aa + 2 * (q * C::kX + 16 * jb * C::PX + 16 * k));
#pragma unroll
          for (int r = 0; r < C::RT; ++r)
            if (C::RT == 1 || jb <= rb + r)
              multiply_planes<C::kIn, C::kIn, 1, C::kFloat>(k & 1 ? w_odd[r] : w[r], x[r], v);
        }
        if (D > 16) {
#pragma unroll
          for (int r = 0; r < C::RT; ++r)
#pragma unroll
            for (int q = 0; q < 8; ++q) w[r][q >> 2][q & 3] += w_odd[r][q >> 2][q & 3];
        }
        uint32_t wp[C::RT][C::kMid][4];
#pragma unroll
        for (int r = 0; r < C::RT; ++r) {
          if (C::RT > 1 && jb > rb + r) continue;
          const bool diagonal = jb == rb + r;
#pragma unroll
          for (int q = 0; q < 8; ++q) {
            const int j = 16 * jb + gc + (q & 1) + (q & 4) * 2;
            const float weight = diagonal ? near[q] : next[q] * far[r];
            w[r][q >> 2][q & 3] *= j >= from[r][(q >> 1) & 1] ? weight : 0.0f;
          }
          if (!diagonal) far[r] *= block_decay;
          split_pair<C::kMid>(w[r][0][0], w[r][0][1], &wp[r][0][0], 4);
          split_pair<C::kMid>(w[r][0][2], w[r][0][3], &wp[r][0][1], 4);
          split_pair<C::kMid>(w[r][1][0], w[r][1][1], &wp[r][0][2], 4);
          split_pair<C::kMid>(w[r][1][2], w[r][1][3], &wp[r][0][3], 4);
        }
#pragma unroll
        for (int t = 0; t < C::OC / 16; t += kGroup) {
          uint32_t v[kGroup][C::kIn][4];
#pragma unroll
          for (int i = 0; i < kGroup; ++i)
#pragma unroll
            for (int q = 0; q < C::kIn; ++q)
              load_matrices_turned(v[i][q], ba + 2 * (q * C::kB + 16 * jb * C::PB + 16 * (t + i)));
#pragma unroll
          for (int r = 0; r < C::RT; ++r)
            if (C::RT == 1 || jb <= rb + r)
              multiply_planes<C::kMid, C::kIn, kGroup, C::kFloat>(&o[r][2 * t], wp[r], v);
        }
      }
#pragma unroll
      for (int r = 0; r < C::RT; ++r)
#pragma unroll
        for (int t = 0; t < C::OC / 8; ++t)
#pragma unroll
          for (int q = 0; q < 4; ++q)
            if (16 * (rb + r) + gr + (q & 2) * 4 < len) bad = fmaf(o[r][t][q], 0.0f, bad);
      if constexpr (C::kColWarps == 1 && sizeof(T) == 2) {
        // to global memory by whole rows, through this warp's rows of x, which nothing reads any more
        __syncwarp();
        __nv_bfloat16* const own = X + 16 * rb * C::PX;
#pragma unroll
        for (int r = 0; r < C::RT; ++r)
#pragma unroll
          for (int half = 0; half < 2; ++half)
#pragma unroll
            for (int t = 0; t < C::OC / 8; ++t)
              *reinterpret_cast<uint32_t*>(own + (16 * r + gr + 8 * half) * C::PX + 8 * t + gc) =
                  pack(o[r][t][2 * half], o[r][t][2 * half + 1]);
        __syncwarp();
#pragma unroll
        for (int e = 0; e < 16 * C::RT / kRowsOut; ++e) {
          const int r = lane / kPieces + e * kRowsOut;
          if (16 * rb + r < len)
            *reinterpret_cast<uint4*>(out_at + ((C::kTurning ? 16 * rb : 0) + e * kRowsOut) * out_step) =
                *reinterpret_cast<const uint4*>(own + r * C::PX + lane % kPieces * kPer);
        }
      } else {
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          const int row = 16 * rb + gr + 8 * half;
          const int64_t i = i0 + row;
          T* const at = static_cast<T*>(s.out) + (s.reverse ? p.t - 1 - i : i) * token_step + int64_t(seq) * D + col + oc + gc;
          if (row < len) {
#pragma unroll
            for (int t = 0; t < C::OC / 8; ++t) {
              const float lo = o[0][t][2 * half], hi = o[0][t][2 * half + 1];
              if constexpr (sizeof(T) == 2)
                *reinterpret_cast<uint32_t*>(at + 8 * t) = pack(lo, hi);
              else
                *reinterpret_cast<float2*>(at + 8 * t) = make_float2(lo, hi);
            }
          }
        }
      }
    }

    __syncwarp();  // behind the stores of a chunk's last rows
    out_at += kChunk * out_step;
    if (!kLocal && C::kTurning) {
      rb = rb + C::RT < C::kRowWarps * C::RT ? rb + C::RT : 0;
      decay_rows();
    }

    // Z <- g^L Z + (l * A)' B, l_j = g^(L - f - j) where no reset lies between token j and the end
    if (holds) {
      bool none = true;
      const int reached = resets ? linked_from(~uint64_t(0), &none) : 0;
      const float through = powers[len];
#pragma unroll
      for (int m = 0; m < C::MT; ++m)
#pragma unroll
        for (int t = 0; t < C::NT; ++t)
#pragma unroll
          for (int q = 0; q < 4; ++q) z[m][t][q] = none ? through * z[m][t][q] : 0.0f;
      const uint32_t at = shared_address(A + ((lane & 7) + (lane >> 4) * 8) * C::PX + ((lane >> 3) & 1) * 8 + srow);
      const uint32_t bt = shared_address(B + (lane & 15) * C::PB + (lane >> 4) * 8 + scol);
#pragma unroll
      for (int j = 0; j < kChunk / 16; ++j) {
        if (j >= live) break;
        float l[4];
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const int i = 16 * j + gc + (q & 1) + (q & 2) * 4;
          l[q] = i >= reached && i < len ? powers[len - f - i] : 0.0f;
        }
        uint32_t key[C::MT][C::kKeys][4];
#pragma unroll
        for (int m = 0; m < C::MT; ++m) {
          float lo[4] = {}, hi[4] = {};
#pragma unroll
          for (int q = C::kIn - 1; q >= 0; --q) {  // the planes' sum is the float32 value again
            uint32_t v[4];
            load_matrices_turned(v, at + 2 * (q * C::kX + 16 * j * C::PX + 16 * m));
#pragma unroll
            for (int u = 0; u < 4; ++u) lo[u] += low_half(v[u]), hi[u] += high_half(v[u]);
          }
#pragma unroll
          for (int u = 0; u < 4; ++u) split_pair<C::kKeys>(l[u & 2] * lo[u], l[(u & 2) + 1] * hi[u], &key[m][0][u], 4);
        }
        constexpr int kGroup = C::NT >= 4 ? 2 : 1;
#pragma unroll
        for (int t = 0; t < C::NT / 2; t += kGroup) {
          uint32_t v[kGroup][C::kIn][4];
#pragma unroll
          for (int i = 0; i < kGroup; ++i)
#pragma unroll
            for (int q = 0; q < C::kIn; ++q)
              load_matrices_turned(v[i][q], bt + 2 * (q * C::kB + 16 * j * C::PB + 16 * (t + i)));
#pragma unroll
          for (int m = 0; m < C::MT; ++m)
            multiply_planes<C::kKeys, C::kIn, kGroup, C::kFloat>(&z[m][2 * t], key[m], v, fine);
        }
      }
    }
    __syncthreads();
  }

#pragma unroll
  for (int m = 0; m < C::MT; ++m)
#pragma unroll
    for (int t = 0; t < C::NT; ++t)
#pragma unroll
      for (int q = 0; q < 4; ++q) bad = fmaf(z[m][t][q], 0.0f, bad);
  float* const end = kLocal ? split.carry + slot * D * D : whole && s.carry_out ? s.carry_out + int64_t(seq) * D * D : nullptr;
  const bool end_turned = !kLocal && s.turned;
  const float end_mul = kLocal ? 1.0f : s.out_mul;
  if (kLocal && threadIdx.x == 0 && col == 0) split.through[slot] = cut ? -1.0f : power(log2_g, last - first);
  // A value that is not finite may have met a masked zero on its way: the definition decides.
  if (__syncthreads_or(bad != bad)) {
    scan_tokens<T, D, DB, C::kThreads, !kLocal>(s, p, n, h, col, first, last, start, turned, start_mul,
                                                reinterpret_cast<float*>(smem), end, end_turned, end_mul);
    return;
  }
  if (end && holds) {
#pragma unroll
    for (int m = 0; m < C::MT; ++m)
#pragma unroll
      for (int t = 0; t < C::NT; ++t)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const int r = srow + 16 * m + gr + (q & 2) * 4, c = col + scol + 8 * t + gc + (q & 1);
          end[end_turned ? c * D + r : r * D + c] = end_mul * z[m][t][q];
        }
  }
}

// The carry at each segment's start from the segments' own, one thread an element.
__global__ void __launch_bounds__(256)
join_kernel(const __grid_constant__ Problem p, const __grid_constant__ Split split, int d) {
  const int64_t size = int64_t(d) * d, sequences = p.n * p.h;
  const int64_t e = int64_t(blockIdx.x) * 256 + threadIdx.x;
  if (e >= p.scans * sequences * size) return;
  const int64_t which = e / size, scan = which / sequences, seq = which % sequences;
  const int at = int(e % size);
  const Scan& s = p.scan[scan];
  const int64_t outside = seq * size + (s.turned ? at % d * d + at / d : at);
  float z = s.carry_in ? s.in_mul * __ldg(s.carry_in + outside) : 0.0f;
  float* const own = split.carry + which * split.segments * size + at;
  const float* const through = split.through + which * split.segments;
  const float g = __ldg(p.decay + seq % p.h);
  constexpr int kAhead = 8;  // loads in flight: the sums are a chain, the loads are not
  for (int64_t g0 = 0; g0 < split.segments; g0 += kAhead) {
    float mine[kAhead], over[kAhead];
#pragma unroll
    for (int i = 0; i < kAhead; ++i)
      if (g0 + i < split.segments) mine[i] = own[(g0 + i) * size], over[i] = through[g0 + i];
#pragma unroll
    for (int i = 0; i < kAhead; ++i)
      if (g0 + i < split.segments) {
        own[(g0 + i) * size] = z;
        // A power of a positive decay that has underflowed leaves an infinity one, as token by token.
        const float kept = over[i] * z;
        z = (over[i] < 0.0f ? 0.0f : kept != kept && z == z && g > 0.0f ? z : kept) + mine[i];
      }
  }
  if (s.carry_out) s.carry_out[outside] = s.out_mul * z;
}

// How a call is split over the time axis. Where the sequences fill more than a quarter of the room on the SMs, not
// at all: the segments' own carries cost a second pass over half of the products (4,096 tokens of bf16 heads of
// 64: 128 sequences 197 us split and 178 whole, 64 sequences 110 and 178, 8 sequences 47 and 176). Else into one
// round of blocks, as many as there is room for at once.
constexpr int64_t kSms = 148;

int64_t split_segments(int64_t t, int64_t blocks, int per_sm, int64_t* per) {
  const int64_t chunks = (t + attn::kChunk - 1) / attn::kChunk, room = kSms * per_sm;
  const int64_t want = blocks > 0 && 4 * blocks <= room ? room / blocks : 1;
  *per = (chunks + want - 1) / want;
  if (*per < 1) *per = 1;
  return chunks > 0 ? (chunks + *per - 1) / *per : 1;
}

struct ScratchSize {
  int64_t t, n, h;
  int scans;
  template <typename T, int D>
  int64_t operator()() const {
    int64_t per;
    const int64_t segments =
        split_segments(t, n * h * scans * (D / attn::Shape<T, D>::DB), attn::Shape<T, D>::kPerSm, &per);
    return segments == 1 ? 0 : scans * n * h * segments * (int64_t(D) * D + 1) * 4;
  }
};

template <typename T, int D>
int launch_scan(const Problem& p, void* scratch, cudaStream_t stream) {
  using C = attn::Shape<T, D>;
  constexpr int kTiles = D / C::DB;
  Split split{};
  const int64_t sequences = p.n * p.h;
  split.segments = split_segments(p.t, sequences * p.scans * kTiles, C::kPerSm, &split.per);
  const int64_t blocks = sequences * p.scans * kTiles * split.segments;
  if (blocks > 0x7fffffff) return RLENV_EINVAL;
  if (cudaError_t e = cudaFuncSetAttribute(chunk_kernel<T, D, false>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmem))
    return int(e);
  if (split.segments > 1) {
    split.carry = static_cast<float*>(scratch);
    split.through = split.carry + p.scans * sequences * split.segments * D * D;
    if (cudaError_t e = cudaFuncSetAttribute(chunk_kernel<T, D, true>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmem))
      return int(e);
    chunk_kernel<T, D, true><<<unsigned(blocks), C::kThreads, C::kSmem, stream>>>(p, split);
    if (const int rc = launch_status()) return rc;
    join_kernel<<<grid_for(p.scans * sequences * D * D, 256), 256, 0, stream>>>(p, split, D);
    if (const int rc = launch_status()) return rc;
  }
  chunk_kernel<T, D, false><<<unsigned(blocks), C::kThreads, C::kSmem, stream>>>(p, split);
  return launch_status();
}

// One token: S <- keep g S + k' v in place, o = scale q S. A block is one head of one environment;
// the state streams through registers once, so the kernel is bound by reading and writing it
// (8 D^2 bytes): 4,096 x 8 heads of 64 in 165 us, 6.6 TB/s. Thread t holds four columns of every
// (kStepThreads * 4 / D)-th row.
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
  __shared__ __align__(16) float part[kRows][D];  // read and written by fours
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

// A few tokens of many sequences, with the state in registers as `step` has it, token after token: bound by reading
// and writing the states (8,000 bfloat16 heads of 64, one token: 55 us, 4.8 TB/s), where a chunk would be mostly
// padding. A state's element (r, c) grows by left_r right_c; a token's results are across_r = scale sum_c (r, c)
// along_c and down_c = scale sum_r (r, c) head_r. Forward, down of k, v and q; dq, across of k, v and do; dk and dv
// from one pass of the adjoint state, across and down of q, do and v, k, last token first. A block is one sequence:
// thread t holds four columns of D / 8 rows. Sums along a row go through the lanes that hold it, half of the values a
// step; those down a column meet in shared memory.
struct Tokens {
  const void *left, *right, *along, *head;
  Strides ls, rs, as, hs;
  const float* decay;
  const uint8_t* resets;
  const float* in;
  float* end;
  void *across, *down;
  float scale, in_mul, out_mul;
  int t, reverse;
  int64_t n, h;
};
constexpr int kMostTokens = 16;

template <int D, bool kAcross, bool kDown>
constexpr int tokens_smem(int t) {
  return t * D * 4 * (2 + (kAcross ? 2 : 0) + (kDown ? 1 + D / 16 : 0));
}

template <typename T, int D, bool kAcross, bool kDown>
__global__ void __launch_bounds__(2 * D) tokens_kernel(const __grid_constant__ Tokens p) {
  constexpr int kLanes = D / 4, kRows = D / 8, kThreads = 2 * D, kWarps = D / 16;
  extern __shared__ __align__(16) unsigned char smem[];
  __shared__ int cut[kMostTokens];
  const int size = p.t * D;
  float* const left = reinterpret_cast<float*>(smem);
  float *const right = left + size, *const along = right + size, *const across = along + size;
  float *const head = right + size + (kAcross ? 2 * size : 0), *const parts = head + size;  // parts: (token, warp, D)
  const int64_t seq = blockIdx.x, n = seq / p.h, h = seq % p.h;
  const int row = threadIdx.x / kLanes * kRows, c = threadIdx.x % kLanes * 4, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  float4 z[kRows];
#pragma unroll
  for (int k = 0; k < kRows; ++k) {
    z[k] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    if (p.in) {
      z[k] = __ldg(reinterpret_cast<const float4*>(p.in + (seq * D + row + k) * D + c));
      z[k].x *= p.in_mul, z[k].y *= p.in_mul, z[k].z *= p.in_mul, z[k].w *= p.in_mul;
    }
  }
  const auto fetch = [&](float* to, const void* from, const Strides& s) {
    const T* at = static_cast<const T*>(from) + n * s.n + h * s.h;
    for (int e = threadIdx.x; e < size; e += kThreads) to[e] = attn::to_float(at[e / D * s.t + e % D]);
  };
  fetch(left, p.left, p.ls);
  fetch(right, p.right, p.rs);
  if (kAcross) fetch(along, p.along, p.as);
  if (kDown) fetch(head, p.head, p.hs);
  if (threadIdx.x < p.t) cut[threadIdx.x] = p.resets ? __ldg(p.resets + threadIdx.x * p.n + n) : 0;
  const float g = __ldg(p.decay + h);
  __syncthreads();
  const auto decay = [&](bool reset) {
#pragma unroll
    for (int k = 0; k < kRows; ++k) {
      z[k].x = reset ? 0.0f : g * z[k].x, z[k].y = reset ? 0.0f : g * z[k].y;
      z[k].z = reset ? 0.0f : g * z[k].z, z[k].w = reset ? 0.0f : g * z[k].w;
    }
  };
  for (int j = 0; j < p.t; ++j) {
    const int i = p.reverse ? p.t - 1 - j : j;
    const bool reset = cut[i] != 0;
    if (!p.reverse) decay(reset);
    const float4 r = *reinterpret_cast<const float4*>(right + i * D + c);
    float4 y = make_float4(0.0f, 0.0f, 0.0f, 0.0f), o = y;
    if (kAcross) y = *reinterpret_cast<const float4*>(along + i * D + c);
    float s[kRows];
#pragma unroll
    for (int k = 0; k < kRows; k += 2) {
      const float2 l = *reinterpret_cast<const float2*>(left + i * D + row + k);
      float2 w = make_float2(0.0f, 0.0f);
      if (kDown) w = *reinterpret_cast<const float2*>(head + i * D + row + k);
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const float lu = u ? l.y : l.x, wu = u ? w.y : w.x;
        float4& v = z[k + u];
        v.x = fmaf(lu, r.x, v.x), v.y = fmaf(lu, r.y, v.y), v.z = fmaf(lu, r.z, v.z), v.w = fmaf(lu, r.w, v.w);
        if (kDown) o.x = fmaf(wu, v.x, o.x), o.y = fmaf(wu, v.y, o.y), o.z = fmaf(wu, v.z, o.z), o.w = fmaf(wu, v.w, o.w);
        if (kAcross) s[k + u] = fmaf(y.x, v.x, fmaf(y.y, v.y, fmaf(y.z, v.z, y.w * v.w)));
      }
    }
    if constexpr (kAcross) {
#pragma unroll
      for (int m = kRows / 2; m >= 1; m /= 2) {  // lanes 2 m apart share their values out
        const bool upper = lane & 2 * m;
#pragma unroll
        for (int k = 0; k < m; ++k) {
          const float give = upper ? s[k] : s[k + m], keep = upper ? s[k + m] : s[k];
          s[k] = keep + __shfl_xor_sync(0xffffffffu, give, 2 * m);
        }
      }
      s[0] += __shfl_xor_sync(0xffffffffu, s[0], 1);
      if (lane % 2 == 0) across[i * D + row + lane % kLanes / 2] = s[0];
    }
    if constexpr (kDown) {
#pragma unroll
      for (int m = kLanes; m < 32; m *= 2) {
        o.x += __shfl_xor_sync(0xffffffffu, o.x, m), o.y += __shfl_xor_sync(0xffffffffu, o.y, m);
        o.z += __shfl_xor_sync(0xffffffffu, o.z, m), o.w += __shfl_xor_sync(0xffffffffu, o.w, m);
      }
      if (lane < kLanes) *reinterpret_cast<float4*>(parts + (i * kWarps + warp) * D + c) = o;
    }
    if (p.reverse) decay(reset);
  }
  if (p.end) {
#pragma unroll
    for (int k = 0; k < kRows; ++k)
      *reinterpret_cast<float4*>(p.end + (seq * D + row + k) * D + c) =
          make_float4(p.out_mul * z[k].x, p.out_mul * z[k].y, p.out_mul * z[k].z, p.out_mul * z[k].w);
  }
  __syncthreads();
  for (int e = threadIdx.x; e < size; e += kThreads) {
    const int64_t at = (e / D * p.n * p.h + seq) * D + e % D;
    if (kAcross) static_cast<T*>(p.across)[at] = attn::from_float<T>(p.scale * across[e]);
    if (kDown) {
      float sum = 0.0f;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) sum += parts[(e / D * kWarps + w) * D + e % D];
      static_cast<T*>(p.down)[at] = attn::from_float<T>(p.scale * sum);
    }
  }
}

template <bool kAcross, bool kDown>
struct TokensRunner {
  const Tokens& p;
  cudaStream_t stream;
  template <typename T, int D>
  int operator()() const {
    constexpr int kMost = tokens_smem<D, kAcross, kDown>(kMostTokens);
    if (kMost > 40 * 1024)
      if (cudaError_t e = cudaFuncSetAttribute(tokens_kernel<T, D, kAcross, kDown>,
                                               cudaFuncAttributeMaxDynamicSharedMemorySize, kMost))
        return int(e);
    tokens_kernel<T, D, kAcross, kDown>
        <<<unsigned(p.n * p.h), 2 * D, tokens_smem<D, kAcross, kDown>(p.t), stream>>>(p);
    return launch_status();
  }
};

bool width_built(int d) { return d == 16 || d == 32 || d == 64 || d == 128; }

// Calls fn<T, D>() for the type and width.
template <typename R, typename F>
R dispatch(int dtype, int d, F&& fn) {
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

bool off_boundary(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 != 0; }

// Rows are read as 16-byte pieces: a base and strides off that boundary are rejected.
bool aligned_rows(const void* p, const int64_t* st, int dtype, int axes) {
  const uint64_t size = dtype == RLENV_F32 ? 4 : 2;
  if (off_boundary(p)) return false;
  for (int i = 0; i < axes; ++i)
    if (uint64_t(st[i]) * size % 16) return false;
  return true;
}

// Whether tokens are taken one after the other: few of them, in as many sequences as give each SM 256 threads.
// Measured in us, this way and by chunks, forward and gradient: bfloat16, 8,000 heads of 64, 1 token 55 and 170, 103
// and 421, 8 tokens 99 and 173, 211 and 427; 2,400 of 128, 8 tokens 175 and 205, 370 and 499; 1,200 of 128, 12
// tokens 137 and 108, 302 and 254; 16,000 of 32, 16 tokens 108 and 99; float32 2,400 heads of 128, 1 token 99
// and 465, 183 and 1,251, 16 tokens 256 and 474, 575 and 1,272; 24,000 of 16, 16 tokens 63 and 153; few sequences,
// 15 of 64, 8 tokens, 5 and 8, 13 and 8; 296 of 16, 8 tokens, 4.4 and 3.8, 9.9 and 7.6.
bool few_tokens(int dtype, int d, int64_t t, int64_t n, int64_t h) {
  return t > 0 && t <= (dtype == RLENV_F32 ? kMostTokens : kMostTokens / 2) && n * h * d >= 128 * 148;
}

struct Runner {
  const Problem& p;
  void* scratch;
  cudaStream_t stream;
  template <typename T, int D>
  int operator()() const { return launch_scan<T, D>(p, scratch, stream); }
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
  return check_sizes(dtype, d, t, n, h, 1.0f) == RLENV_OK ? dispatch<int64_t>(dtype, d, ScratchSize{t, n, h, backward ? 3 : 1}) : -1;
}

int rlenv_linear_attention_forward(int dtype, int d, int64_t t, int64_t n, int64_t h, const void* q, const void* k,
                                   const void* v, const int64_t* strides, const float* decay, const uint8_t* resets,
                                   float scale, const float* state_in, void* out, float* state_out, void* scratch,
                                   int64_t scratch_bytes, void* stream) {
  using namespace rlenv;
  if (const int rc = check_sizes(dtype, d, t, n, h, scale)) return rc;
  if (n == 0 || h == 0) return RLENV_OK;
  if (t > 0 && (!q || !k || !v || !strides || !out || off_boundary(out))) return RLENV_EINVAL;
  if (!decay || !state_out || state_in == state_out) return RLENV_EINVAL;
  static const int64_t kNone[9] = {};
  const int64_t* st = t > 0 ? strides : kNone;
  if (!aligned_rows(q, st, dtype, 3) || !aligned_rows(k, st + 3, dtype, 3) || !aligned_rows(v, st + 6, dtype, 3))
    return RLENV_EINVAL;
  if (!scratch_holds(scratch, scratch_bytes, dispatch<int64_t>(dtype, d, ScratchSize{t, n, h, 1}))) return RLENV_EINVAL;
  if (few_tokens(dtype, d, t, n, h) && !off_boundary(state_in) && !off_boundary(state_out)) {
    const Tokens f{k, v, nullptr, q, {st[3], st[4], st[5]}, {st[6], st[7], st[8]}, {}, {st[0], st[1], st[2]}, decay,
                   resets, state_in, state_out, nullptr, out, scale, 1.0f, 1.0f, int(t), 0, n, h};
    return dispatch<int>(dtype, d, TokensRunner<false, true>{f, as_stream(stream)});
  }
  Problem p{};
  p.t = t, p.n = n, p.h = h, p.decay = decay, p.resets = resets, p.scale = scale, p.scans = 1;
  p.scan[0] = Scan{q, k, v, {st[0], st[1], st[2]}, {st[3], st[4], st[5]}, {st[6], st[7], st[8]},
                   out, state_in, state_out, 1.0f, 1.0f, 0, 0};
  return dispatch<int>(dtype, d, Runner{p, scratch, as_stream(stream)});
}

int rlenv_linear_attention_backward(int dtype, int d, int64_t t, int64_t n, int64_t h, const void* grad_out,
                                    const void* q, const void* k, const void* v, const int64_t* strides,
                                    const float* decay, const uint8_t* resets, float scale, const float* state_in,
                                    const float* grad_state_out, void* grad_q, void* grad_k, void* grad_v,
                                    float* grad_state_in, void* scratch, int64_t scratch_bytes, void* stream) {
  using namespace rlenv;
  if (const int rc = check_sizes(dtype, d, t, n, h, scale)) return rc;
  if (n == 0 || h == 0) return RLENV_OK;
  if (t > 0 && (!grad_out || !q || !k || !v || !strides || !grad_q || !grad_k || !grad_v ||
                off_boundary(grad_q) || off_boundary(grad_k) || off_boundary(grad_v)))
    return RLENV_EINVAL;
  if (!decay || (grad_state_in && grad_state_in == grad_state_out)) return RLENV_EINVAL;
  static const int64_t kNone[12] = {};
  const int64_t* st = t > 0 ? strides : kNone;
  if (!aligned_rows(grad_out, st, dtype, 3) || !aligned_rows(q, st + 3, dtype, 3) ||
      !aligned_rows(k, st + 6, dtype, 3) || !aligned_rows(v, st + 9, dtype, 3))
    return RLENV_EINVAL;
  if (!scratch_holds(scratch, scratch_bytes, dispatch<int64_t>(dtype, d, ScratchSize{t, n, h, 3}))) return RLENV_EINVAL;
  const Strides ds{st[0], st[1], st[2]}, qs{st[3], st[4], st[5]}, ks{st[6], st[7], st[8]}, vs{st[9], st[10], st[11]};
  // The reverse scans carry R / scale, so that the common factor stays outside.
  const float inv = 1.0f / scale;
  if (few_tokens(dtype, d, t, n, h) && !off_boundary(state_in) && !off_boundary(grad_state_out) && !off_boundary(grad_state_in)) {
    const Tokens f{k, v, grad_out, nullptr, ks, vs, ds, {}, decay, resets, state_in, nullptr, grad_q, nullptr, scale,
                   1.0f, 1.0f, int(t), 0, n, h};
    if (const int rc = dispatch<int>(dtype, d, TokensRunner<true, false>{f, as_stream(stream)})) return rc;
    const Tokens r{q, grad_out, v, k, qs, ds, vs, ks, decay, resets, grad_state_out, grad_state_in, grad_k, grad_v,
                   scale, inv, scale, int(t), 1, n, h};
    return dispatch<int>(dtype, d, TokensRunner<true, true>{r, as_stream(stream)});
  }
  Problem p{};
  p.t = t, p.n = n, p.h = h, p.decay = decay, p.resets = resets, p.scale = scale, p.scans = 3;
  p.scan[0] = Scan{grad_out, v, k, ds, vs, ks, grad_q, state_in, nullptr, 1.0f, 1.0f, 1, 0};
  p.scan[1] = Scan{v, grad_out, q, vs, ds, qs, grad_k, grad_state_out, nullptr, inv, scale, 1, 1};
  p.scan[2] = Scan{k, q, grad_out, ks, qs, ds, grad_v, grad_state_out, grad_state_in, inv, scale, 0, 1};
  return dispatch<int>(dtype, d, Runner{p, scratch, as_stream(stream)});
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
  return dispatch<int>(dtype, d,
                  StepRunner{q, k, v, {0, strides[0], strides[1]}, {0, strides[2], strides[3]},
                             {0, strides[4], strides[5]}, decay, resets, scale, n, h, state, out, as_stream(stream)});
}
