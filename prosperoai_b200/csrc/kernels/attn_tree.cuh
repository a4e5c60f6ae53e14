// Attention of drafted nodes over a cache view (pai_b200_attn_tree_f16kv): what its kernels share.
//
// A sequence's query rows are its nodes times the G = h / kv_heads query heads
// that share a kv head, in tiles of MR rows. Every row tile of every kv head
// ("unit") goes over the same keys: the committed positions, then the nodes
// themselves, in tiles of KT positions, with one running softmax.
//
//   s_j = (q . k_j) / sqrt(hd) if row sees j, else -inf
//   m = max s_j, l = sum e^(s_j - m), o = sum e^(s_j - m) v_j / l
//
// Work split: the (unit, tile) pairs of all sequences, in order, are cut into
// gridDim.x even ranges, whatever the lengths are (they are known on the
// device only). A CTA writes the units that lie in its range to `out`, and
// (o, m, l) of a unit that it shares to scratch; the parts of such a unit are
// joined in order, so that the result does not depend on which CTA is last.
//
// Arithmetic: K and V are fp16 as stored. q, scaled by a power of two for
// each row, and the softmax weights are split into an fp16 part and an fp16
// remainder and multiplied twice, with fp32 sums. Both parts are rounded, so
// an element is off by 2^-22 of itself, or by half of fp16's smallest step,
// 2^-25, whichever is more. A row's largest element of q lies at 2^14 or
// above: what is below 2^-17 of it is off by 2^-39 of it at most. The weights
// carry a factor 2^12: those below 2^-15 of the largest are off by 2^-37 of it.
#pragma once
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include "../b200_internal.h"
#include "b200_device.cuh"
#include "kv_view.cuh"

namespace {

constexpr uint32_t kMaxSeqs = 1024;
constexpr float kPShift = 12.0f;  // weights carry 2^12

struct TreeParams {
  KvDev c;
  uint32_t h, g, max_nodes, words, max_blocks;  // g: query heads of a kv head; max_blocks: row tiles of a sequence
  uint64_t rows;
  const int32_t *lens, *off;
  const uint64_t *mask;
  const float *q;
  float *out;
  float *part_o;   // scratch [2 gridDim.x][MR][hd]
  float *part_ml;  // scratch [2 gridDim.x][MR][2]
  uint32_t *cnt;   // counters [n_seq][kv head][row tile], left at zero
  uint32_t *units; // scratch [n_seq][kv head][row tile][2]: parts of a unit, slot of the first
  uint32_t slots;  // parts that the scratch holds, two a CTA
  uint32_t *err;
  uint64_t wait_ns;
  uint32_t chunk;  // tcgen05 form: positions of one tensor copy
  float scale;     // log2(e) / sqrt(hd): multiplies q, so that scores are exponents of two but for a power of two
};

// (x, y) -> packed fp16 parts and packed fp16 remainders
__device__ __forceinline__ void split_f16(float x, float y, uint32_t &hi, uint32_t &lo) {
  const __half2 h = __floats2half2_rn(x, y);
  const float2 f = __half22float2(h);
  const __half2 l = __floats2half2_rn(x - f.x, y - f.y);
  hi = *reinterpret_cast<const uint32_t *>(&h);
  lo = *reinterpret_cast<const uint32_t *>(&l);
}

// 2^x of the special function unit: 2^-22 relative, results below 2^-126 are 0
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// What a row's scores are taken relative to, from their maximum: 2^12 times the weights. Rounded up, so that no weight is
// above 2^12 where a score's steps are larger than 12 (rounded to nearest, 2^26 - 12 is 2^26 - 16, and 2^16 is no fp16).
__device__ __forceinline__ float shifted(float top) { return __fsub_ru(top, kPShift); }

// Bits [at, at + 64) of a row of `words` 64-bit words; at may be negative.
__device__ __forceinline__ uint64_t window(const uint64_t *m, uint32_t words, int32_t at) {
  const int32_t w = at >> 6, sh = at & 63;
  const uint64_t a = w >= 0 && w < (int32_t)words ? m[w] : 0;
  const uint64_t b = w + 1 >= 0 && w + 1 < (int32_t)words ? m[w + 1] : 0;
  return sh ? (a >> sh) | (b << (64 - sh)) : a;
}
// The lowest n bits (n below 0: none; above 63: all).
__device__ __forceinline__ uint64_t low_bits(int64_t n) {
  return n <= 0 ? 0 : n >= 64 ? ~0ull : (1ull << n) - 1;
}

// Where part q of a unit lies whose first part lies in slot `first`: the other parts are the first ones of their CTAs.
__host__ __device__ __forceinline__ uint32_t part_slot(uint32_t first, uint32_t q) {
  return q == 0 ? first : (first & ~1u) + 2 * q;
}
// How many parts a unit's entry names, 0 where they would lie outside the scratch. After a wait has run out in some CTA
// its other units have no entry, and what lies there instead is whatever the scratch held before.
__host__ __device__ __forceinline__ uint32_t unit_parts(uint32_t parts, uint32_t first, uint32_t slots) {
  if (parts == 0 || parts > slots || first >= slots) return 0;
  return part_slot(first, parts - 1) < slots ? parts : 0;
}

// One sequence's share of the work.
struct SeqWork {
  uint32_t len, nodes, first, blocks, tiles;
};
template <uint32_t MR, uint32_t KT>
__device__ __forceinline__ SeqWork seq_work(const TreeParams &p, uint32_t s) {
  SeqWork w;
  w.nodes = kv_nodes(p.off, s, p.rows, p.max_nodes, &w.first);
  w.len = kv_len(p.c, p.lens, s);
  w.blocks = (w.nodes * p.g + MR - 1) / MR;
  w.tiles = (w.len + w.nodes + KT - 1) / KT;
  return w;
}

// upto[s]: (unit, tile) pairs of the sequences before s. Every thread of the block calls it; a barrier must follow.
template <uint32_t MR, uint32_t KT, uint32_t THREADS>
__device__ __forceinline__ void pairs_before(const TreeParams &p, uint64_t *upto) {
  const uint32_t n_seq = p.c.n_seq, lane = threadIdx.x & 31;
  for (uint32_t s = threadIdx.x; s < n_seq; s += THREADS) {
    const SeqWork w = seq_work<MR, KT>(p, s);
    upto[s + 1] = (uint64_t)w.blocks * w.tiles * p.c.hk;
  }
  if (threadIdx.x == 0) upto[0] = 0;
  __syncthreads();
  if (threadIdx.x < 32) {
    uint64_t sum = 0;
    for (uint32_t s0 = 0; s0 < n_seq; s0 += 32) {
      const uint32_t s = s0 + lane;
      uint64_t x = s < n_seq ? upto[s + 1] : 0;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const uint64_t y = __shfl_up_sync(0xffffffffu, x, o);
        if (lane >= (uint32_t)o) x += y;
      }
      x += sum;
      if (s < n_seq) upto[s + 1] = x;
      sum = __shfl_sync(0xffffffffu, x, 31);
    }
  }
}

// 2^-e (down) that brings a row's largest element `top` into [2^14, 2^15), the most that fp16 holds with a bit to spare, and
// 2^e (up); 1 for a row that is not finite. (Rows of elements below 2^-112 stay smaller, so that 2^e is no subnormal.) With
// [1, 2) instead, a row with one element of 1024 times the others' size against a K channel as much smaller was 3e-5 off.
__device__ __forceinline__ void row_scale(float top, float &down, float &up) {
  const uint32_t ex = __float_as_uint(top) >> 23, e = ex < 15 ? 15 : ex;
  down = ex < 255 ? __uint_as_float((268 - e) << 23) : 1.0f;
  up = ex < 255 ? __uint_as_float((e - 14) << 23) : 1.0f;
}

}  // namespace
