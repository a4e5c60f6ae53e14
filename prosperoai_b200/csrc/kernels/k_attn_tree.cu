// Attention of drafted nodes over a cache view (pai_b200_attn_tree_f16kv).
//
// A sequence's query rows are its nodes times the G = h / kv_heads query heads
// that share a kv head, in tiles of MR rows. Every row tile of every kv head
// ("unit") goes over the same keys: the committed positions, then the nodes
// themselves, in tiles of kTile positions, with one running softmax.
//
//   s_j = (q . k_j) / sqrt(hd) if row sees j, else -inf
//   m = max s_j, l = sum e^(s_j - m), o = sum e^(s_j - m) v_j / l
//
// Work split: the (unit, tile) pairs of all sequences, in order, are cut into
// gridDim.x even ranges, whatever the lengths are (they are known on the
// device only). A CTA writes the units that lie in its range to `out`, and
// (o, m, l) of a unit that it shares to scratch; the last CTA of such a unit
// joins the parts in order, so that the result does not depend on which CTA
// is last.
//
// Arithmetic: K and V are fp16 as stored. q, scaled by a power of two for
// each row, and the softmax weights are split into an fp16 part and an fp16
// remainder and multiplied twice, with fp32 sums: 22 bits of each, so that
// the products are as exact as fp32 ones. The weights carry a factor 2^12
// that keeps the remainders of small ones above fp16's smallest step.
#include <cuda.h>  // CUtensorMap and its enums (types only; the encoder comes from the runtime)
#include <cudaTypedefs.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>

#include "../b200_internal.h"
#include "b200_device.cuh"
#include "kv_view.cuh"

namespace {

constexpr uint32_t kTile = 64, kThreads = 128, kMaxSeqs = 1024;
constexpr uint32_t kGrid = 296;  // two CTAs an SM
constexpr int kStages = 3;
constexpr float kPShift = 12.0f;

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
  uint32_t *err;
  uint64_t wait_ns;
  uint32_t chunk;  // tcgen05 form: positions of one tensor copy
  float scale;     // log2(e) / sqrt(hd)
};

__device__ __forceinline__ void mma_f16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
      "{%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], const void *p) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(smem_u32(p)));
}
__device__ __forceinline__ void ldsm4t(uint32_t (&r)[4], const void *p) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(smem_u32(p)));
}
// 16 bytes global -> shared; `ok` false writes zeros and reads nothing
__device__ __forceinline__ void cp16(void *dst, const void *src, bool ok) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(dst)), "l"(src), "r"(ok ? 16u : 0u)
               : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
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

// 2^-e (down) that brings a row's largest element `top` into [1, 2), and 2^e; 1 for a row of zeros, subnormals or
// infinities.
__device__ __forceinline__ void row_scale(float top, float &down, float &up) {
  const uint32_t ex = __float_as_uint(top) >> 23;
  const bool turn = ex >= 1 && ex <= 252;
  down = turn ? __uint_as_float((254 - ex) << 23) : 1.0f;
  up = turn ? __uint_as_float(ex << 23) : 1.0f;
}

// Shared memory of a stage: K then V rows, padded so that the eight rows of an ldmatrix lie in different banks.
template <int HD>
struct Stage {
  __half k[kTile][HD + 8];
  __half v[kTile][HD + 8];
};

// Join the parts of a unit: CTAs c0 .. c0 + parts - 1, in order. First every row's maximum, weights 2^(m - max) and
// sum, in shared memory `ws` [MR][parts]; then the outputs, 8 parts' loads in flight.
template <int HD, uint32_t MR>
__device__ __noinline__ void join_parts(const TreeParams &p, const SeqWork &w, uint32_t kvh, uint32_t block, uint64_t c0,
                                        uint32_t parts, uint64_t unit0, uint64_t all, uint64_t grid, float *ws) {
  const uint32_t t = threadIdx.x, lane = t & 31, warp = t >> 5;
  const uint32_t rows = min(MR, w.nodes * p.g - block * MR);
  // the unit is the first of a CTA's range, or the last; only CTA c0's range can begin before it
  const bool late = c0 * all / grid < unit0;
  auto slot = [&](uint32_t q) { return 2 * (c0 + q) + (q == 0 && late); };
  float *inv = ws + MR * parts;
  for (uint32_t r = warp; r < rows; r += kThreads / 32) {
    float M = -INFINITY;
    for (uint32_t q = lane; q < parts; q += 32) {
      const float mq = __ldcg(&p.part_ml[(slot(q) * MR + r) * 2]);
      ws[r * parts + q] = mq;
      M = fmaxf(M, mq);
    }
    M = warp_max(M);
    float L = 0.0f;
    for (uint32_t q = lane; q < parts; q += 32) {
      const float mq = ws[r * parts + q], e = mq == -INFINITY ? 0.0f : ex2(mq - M);
      L += __ldcg(&p.part_ml[(slot(q) * MR + r) * 2 + 1]) * e;
      ws[r * parts + q] = e;
    }
    L = warp_sum(L);
    if (lane == 0) inv[r] = L != 0.0f ? 1.0f / L : 0.0f;
  }
  __syncthreads();
  for (uint32_t e = t; e < rows * (HD / 4); e += kThreads) {
    const uint32_t r = e / (HD / 4), d = (e % (HD / 4)) * 4;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    for (uint32_t q0 = 0; q0 < parts; q0 += 8) {
      float4 f[8];
#pragma unroll
      for (int u = 0; u < 8; u++)
        if (q0 + u < parts) f[u] = __ldcg(reinterpret_cast<const float4 *>(p.part_o + (slot(q0 + u) * MR + r) * HD + d));
#pragma unroll
      for (int u = 0; u < 8; u++)
        if (q0 + u < parts) {
          const float y = ws[r * parts + q0 + u];
          acc.x = fmaf(f[u].x, y, acc.x), acc.y = fmaf(f[u].y, y, acc.y);
          acc.z = fmaf(f[u].z, y, acc.z), acc.w = fmaf(f[u].w, y, acc.w);
        }
    }
    const uint32_t rr = block * MR + r;
    const float y = inv[r];
    *reinterpret_cast<float4 *>(p.out + ((size_t)(w.first + rr / p.g) * p.h + kvh * p.g + rr % p.g) * HD + d) =
        make_float4(acc.x * y, acc.y * y, acc.z * y, acc.w * y);
  }
}

// WM warps share a tile's rows (16 each), 4 / WM share its positions.
template <int HD, int WM>
__global__ void __launch_bounds__(kThreads, 2) k_attn_tree(TreeParams p) {
  constexpr uint32_t MR = 16 * WM, WN = 4 / WM, NT = 8 / WN, CH = HD / 8;
  extern __shared__ __align__(16) uint8_t smem[];
  Stage<HD> *st = reinterpret_cast<Stage<HD> *>(smem);
  __shared__ uint64_t upto[kMaxSeqs + 1];
  __shared__ int64_t where[4][kTile];             // element offsets of the rows of the next tiles, -1: none
  __shared__ __align__(8) uint32_t valid[4][2];   // their positions that hold a row
  __shared__ uint64_t odd;                        // nodes of a tile with a non-finite V row
  __shared__ uint32_t ticket;
  const uint32_t t = threadIdx.x, lane = t & 31, warp = t >> 5, wm = warp % WM, wn = warp / WM;
  const uint32_t gq = lane >> 2, tq = lane & 3;
  const uint32_t n_seq = p.c.n_seq, hk = p.c.hk;
  pdl_trigger();
  pdl_wait();

  pairs_before<MR, kTile, kThreads>(p, upto);
  __syncthreads();
  const uint64_t all = upto[n_seq], cta = blockIdx.x, grid = gridDim.x < all ? gridDim.x : all;
  if (cta >= grid) return;  // every CTA of the cut has at least one pair
  uint64_t at = cta * all / grid;
  const uint64_t end = (cta + 1) * all / grid, begin = at;
  uint32_t s = 0;
  for (uint32_t lo = 0, hi = n_seq; at < end && lo < hi;) {  // the sequence of the first pair
    const uint32_t mid = (lo + hi) / 2;
    if (upto[mid + 1] <= at) lo = mid + 1; else hi = mid;
    s = lo;
  }

  while (at < end) {
    while (upto[s + 1] <= at) s++;
    const SeqWork w = seq_work<MR, kTile>(p, s);
    const uint64_t unit = (at - upto[s]) / w.tiles, unit0 = upto[s] + unit * w.tiles, unit1 = unit0 + w.tiles;
    const uint32_t kvh = (uint32_t)(unit / w.blocks), block = (uint32_t)(unit % w.blocks);
    const uint32_t tile0 = (uint32_t)(at - unit0), tile1 = (uint32_t)((end < unit1 ? end : unit1) - unit0);
    const uint32_t total = w.len + w.nodes;
    const __half *kp = p.c.k + (size_t)kvh * p.c.head_stride, *vp = p.c.v + (size_t)kvh * p.c.head_stride;

    // this thread's two rows: node, query head, q fragments (part and remainder), factor of its scores
    uint32_t node[2];
    float factor[2];
    bool live[2];
    uint32_t qh[HD / 16][4], ql[HD / 16][4];
#pragma unroll
    for (int x = 0; x < 2; x++) {
      const uint32_t r = block * MR + wm * 16 + gq + 8 * x;
      node[x] = r / p.g;
      live[x] = node[x] < w.nodes;
      const float *qr = p.q + ((size_t)(w.first + (live[x] ? node[x] : 0)) * p.h + kvh * p.g + r % p.g) * HD;
      float top = 0.0f;
#pragma unroll
      for (int k = 0; k < HD / 16; k++)
#pragma unroll
        for (int e = 0; e < 2; e++) {
          const float2 f = live[x] ? *reinterpret_cast<const float2 *>(qr + 16 * k + 8 * e + 2 * tq) : make_float2(0.f, 0.f);
          qh[k][x + 2 * e] = __float_as_uint(f.x);
          ql[k][x + 2 * e] = __float_as_uint(f.y);
          top = fmaxf(top, fmaxf(fabsf(f.x), fabsf(f.y)));
        }
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
      float down, up;
      row_scale(top, down, up);
      factor[x] = p.scale * up;
#pragma unroll
      for (int k = 0; k < HD / 16; k++)
#pragma unroll
        for (int e = 0; e < 2; e++) {
          uint32_t &a = qh[k][x + 2 * e], &b = ql[k][x + 2 * e];
          split_f16(__uint_as_float(a) * down, __uint_as_float(b) * down, a, b);
        }
    }

    float o[HD / 8][4];
#pragma unroll
    for (int n = 0; n < HD / 8; n++) o[n][0] = o[n][1] = o[n][2] = o[n][3] = 0.0f;
    float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f};

    // Row offsets are looked up (page table, a division) one tile before the copies that use them, one row a
    // thread; the copies of tile n + 2 are issued while tile n is multiplied.
    auto find = [&](uint32_t tile) -> int64_t {
      const uint32_t pos = tile * kTile + t;
      return t < kTile && tile < tile1 && pos < total ? kv_row(p.c, s, pos) : -1;
    };
    auto note = [&](uint32_t n, int64_t at_row) {
      if (t < kTile) {
        where[n % 4][t] = at_row;
        const uint32_t bits = __ballot_sync(0xffffffffu, at_row >= 0);
        if (lane == 0) valid[n % 4][warp] = bits;
      }
    };
    auto load = [&](uint32_t n) {
      Stage<HD> &sg = st[n % kStages];
      const int64_t *wh = where[n % 4];
#pragma unroll
      for (uint32_t i = 0; i < kTile * CH / kThreads; i++) {
        const uint32_t r = t / CH + i * (kThreads / CH), ch = t % CH;
        const int64_t at_row = wh[r];
        const bool ok = at_row >= 0;
        cp16(&sg.k[r][ch * 8], kp + (ok ? at_row : 0) + ch * 8, ok);
        cp16(&sg.v[r][ch * 8], vp + (ok ? at_row : 0) + ch * 8, ok);
      }
    };

    __syncthreads();  // the stages are free
#pragma unroll
    for (uint32_t i = 0; i < 3; i++) note(i, find(tile0 + i));
    __syncthreads();
    for (uint32_t i = 0; i < 2; i++) {
      if (tile0 + i < tile1) load(i);
      cp_commit();
    }
    for (uint32_t tile = tile0; tile < tile1; tile++) {
      const uint32_t n = tile - tile0;
      cp_wait<kStages - 2>();
      __syncthreads();  // this tile has landed, the last one's stage is free, the offsets of tile n + 2 are there
      if (tile + 2 < tile1) load(n + 2);
      cp_commit();
      const int64_t ahead = find(tile + 3);
      const bool drafted = (tile + 1) * kTile > w.len;  // the tile holds nodes
      Stage<HD> &sg = st[n % kStages];
      if (drafted) {
        // A non-finite V row may only reach the rows that see its node, and a weight of
        // 0 does not keep it out of a product: such elements become 0 here and are
        // added below where they are seen.
        if (t == 0) odd = 0;
        __syncthreads();
        for (uint32_t e = t; e < kTile * CH; e += kThreads) {
          uint4 &c4 = *reinterpret_cast<uint4 *>(&sg.v[e / CH][(e % CH) * 8]);
          uint32_t *cw = reinterpret_cast<uint32_t *>(&c4);
          bool bad = false;
#pragma unroll
          for (int i = 0; i < 4; i++) {
            if ((cw[i] & 0x7C00u) == 0x7C00u) cw[i] &= 0xFFFF0000u, bad = true;
            if ((cw[i] & 0x7C000000u) == 0x7C000000u) cw[i] &= 0xFFFFu, bad = true;
          }
          if (bad) atomicOr((unsigned long long *)&odd, 1ull << (e / CH));
        }
        __syncthreads();
      }
      const uint64_t rows_ok = *reinterpret_cast<const uint64_t *>(valid[n % 4]);
      const bool masked = drafted || rows_ok != ~0ull;
      uint64_t sees[2] = {rows_ok, rows_ok};
      if (drafted) {
        const int32_t base = (int32_t)(tile * kTile - w.len);  // node of the tile's first position
#pragma unroll
        for (int x = 0; x < 2; x++) {
          uint64_t b = low_bits(-(int64_t)base);
          if (live[x])
            b |= p.mask ? window(p.mask + (size_t)(w.first + node[x]) * p.words, p.words, base) & ~low_bits(-(int64_t)base)
                        : low_bits((int64_t)node[x] + 1 - base);
          sees[x] &= b;
        }
      }

      // S = q K^T of this warp's NT x 8 positions
      float sc[NT][4];
#pragma unroll
      for (uint32_t nt = 0; nt < NT; nt++) sc[nt][0] = sc[nt][1] = sc[nt][2] = sc[nt][3] = 0.0f;
#pragma unroll
      for (int k = 0; k < HD / 32; k++)
#pragma unroll
        for (uint32_t nt = 0; nt < NT; nt++) {
          uint32_t b[4];
          ldsm4(b, &sg.k[(wn * NT + nt) * 8 + (lane & 7)][32 * k + 8 * (lane >> 3)]);
          mma_f16(sc[nt], qh[2 * k], b[0], b[1]);
          mma_f16(sc[nt], ql[2 * k], b[0], b[1]);
          mma_f16(sc[nt], qh[2 * k + 1], b[2], b[3]);
          mma_f16(sc[nt], ql[2 * k + 1], b[2], b[3]);
        }
      // scores in powers of two, unseen ones -inf, running maximum of a row (its 4 threads share it)
      float mt[2] = {-INFINITY, -INFINITY};
#pragma unroll
      for (uint32_t nt = 0; nt < NT; nt++)
#pragma unroll
        for (int e = 0; e < 4; e++) {
          const int x = e >> 1;
          sc[nt][e] *= factor[x];
          if (masked) {
            const uint32_t j = (wn * NT + nt) * 8 + 2 * tq + (e & 1);
            if (!((sees[x] >> j) & 1)) sc[nt][e] = -INFINITY;
          }
          mt[x] = fmaxf(mt[x], sc[nt][e]);
        }
      float corr[2], sub[2];
#pragma unroll
      for (int x = 0; x < 2; x++) {
        mt[x] = fmaxf(mt[x], __shfl_xor_sync(0xffffffffu, mt[x], 1));
        mt[x] = fmaxf(mt[x], __shfl_xor_sync(0xffffffffu, mt[x], 2));
        const float mn = fmaxf(m[x], mt[x]);
        corr[x] = m[x] == mn ? 1.0f : ex2(m[x] - mn);
        m[x] = mn;
        sub[x] = mn == -INFINITY ? 0.0f : mn - kPShift;
        l[x] *= corr[x];
      }
      // weights as A fragments
      uint32_t ph[NT / 2][4], pl[NT / 2][4];
#pragma unroll
      for (uint32_t ks = 0; ks < NT / 2; ks++)
#pragma unroll
        for (int y = 0; y < 2; y++) {
          float pv[4];
#pragma unroll
          for (int e = 0; e < 4; e++) {
            pv[e] = ex2(sc[2 * ks + y][e] - sub[e >> 1]);
            l[e >> 1] += pv[e];
          }
          split_f16(pv[0], pv[1], ph[ks][2 * y], pl[ks][2 * y]);
          split_f16(pv[2], pv[3], ph[ks][2 * y + 1], pl[ks][2 * y + 1]);
        }
      // O = O corr + P V. The tensor cores cut off what an accumulator cannot hold, always towards zero: over
      // thousands of tiles that adds up (5e-5 of the output at 32768 positions). So they sum one tile, from
      // zero, and the tiles are added by rounding additions (2e-7).
#pragma unroll
      for (int n2 = 0; n2 < HD / 16; n2++) {
        float d0[4] = {0.f, 0.f, 0.f, 0.f}, d1[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (uint32_t ks = 0; ks < NT / 2; ks++) {
          uint32_t b[4];
          ldsm4t(b, &sg.v[wn * (NT * 8) + 16 * ks + (lane & 15)][16 * n2 + 8 * (lane >> 4)]);
          mma_f16(d0, ph[ks], b[0], b[1]);
          mma_f16(d1, ph[ks], b[2], b[3]);
          mma_f16(d0, pl[ks], b[0], b[1]);
          mma_f16(d1, pl[ks], b[2], b[3]);
        }
#pragma unroll
        for (int e = 0; e < 4; e++) {
          o[2 * n2][e] = fmaf(o[2 * n2][e], corr[e >> 1], d0[e]);
          o[2 * n2 + 1][e] = fmaf(o[2 * n2 + 1][e], corr[e >> 1], d1[e]);
        }
      }
      if (drafted && odd) {
        // the non-finite elements of nodes in this warp's positions, for the rows that see them
        for (uint64_t left = odd & (low_bits((wn + 1) * NT * 8) & ~low_bits(wn * NT * 8)); left; left &= left - 1) {
          const uint32_t j = __ffsll((long long)left) - 1;
          const int64_t at_row = kv_row(p.c, s, tile * kTile + j);
#pragma unroll
          for (int n2 = 0; n2 < HD / 8; n2++) {
            const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(vp + at_row + 8 * n2 + 2 * tq));
#pragma unroll
            for (int x = 0; x < 2; x++)
              if ((sees[x] >> j) & 1) {
                if (!isfinite(f.x)) o[n2][2 * x] += f.x;
                if (!isfinite(f.y)) o[n2][2 * x + 1] += f.y;
              }
          }
        }
      }
      note(n + 3, ahead);
    }
    cp_wait<0>();
    // row sums: each of a row's 4 threads holds a part
#pragma unroll
    for (int x = 0; x < 2; x++) {
      l[x] += __shfl_xor_sync(0xffffffffu, l[x], 1);
      l[x] += __shfl_xor_sync(0xffffffffu, l[x], 2);
    }
    __syncthreads();
    // the warps that share rows join over their positions: o, m and l in shared memory (the stages are free)
    float *so = reinterpret_cast<float *>(smem);            // [WN][MR][HD + 4]
    float *sm = so + WN * MR * (HD + 4);                    // [WN][MR][2]
    constexpr uint32_t OS = HD + 4;
#pragma unroll
    for (int x = 0; x < 2; x++) {
      const uint32_t r = wm * 16 + gq + 8 * x;
      float *d = so + (wn * MR + r) * OS + 2 * tq;
#pragma unroll
      for (int n2 = 0; n2 < HD / 8; n2++)
        *reinterpret_cast<float2 *>(d + 8 * n2) = make_float2(o[n2][2 * x], o[n2][2 * x + 1]);
      if (tq == 0) {
        sm[(wn * MR + r) * 2] = m[x];
        sm[(wn * MR + r) * 2 + 1] = l[x];
      }
    }
    __syncthreads();
    const bool whole = tile0 == 0 && tile1 == w.tiles;
    const uint64_t slot = 2 * cta + (begin >= unit0 ? 0 : 1);
    for (uint32_t e = t; e < MR * (HD / 4); e += kThreads) {
      const uint32_t r = e / (HD / 4), d = (e % (HD / 4)) * 4;
      float M = -INFINITY;
#pragma unroll
      for (uint32_t y = 0; y < WN; y++) M = fmaxf(M, sm[(y * MR + r) * 2]);
      float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
      float L = 0.0f;
#pragma unroll
      for (uint32_t y = 0; y < WN; y++) {
        const float my = sm[(y * MR + r) * 2], wy = my == -INFINITY ? 0.0f : ex2(my - M);
        if (my == -INFINITY) continue;
        const float4 f = *reinterpret_cast<const float4 *>(so + (y * MR + r) * OS + d);
        acc.x = fmaf(f.x, wy, acc.x), acc.y = fmaf(f.y, wy, acc.y);
        acc.z = fmaf(f.z, wy, acc.z), acc.w = fmaf(f.w, wy, acc.w);
        L = fmaf(sm[(y * MR + r) * 2 + 1], wy, L);
      }
      const uint32_t rr = block * MR + r, nd = rr / p.g;
      if (whole) {
        if (nd < w.nodes) {
          const float inv = L != 0.0f ? 1.0f / L : 0.0f;  // a row that sees nothing gets zeros
          *reinterpret_cast<float4 *>(p.out + ((size_t)(w.first + nd) * p.h + kvh * p.g + rr % p.g) * HD + d) =
              make_float4(acc.x * inv, acc.y * inv, acc.z * inv, acc.w * inv);
        }
      } else {
        *reinterpret_cast<float4 *>(p.part_o + (slot * MR + r) * HD + d) = acc;
        if (d == 0) {
          p.part_ml[(slot * MR + r) * 2] = M;
          p.part_ml[(slot * MR + r) * 2 + 1] = L;
        }
      }
    }
    if (!whole) {
      // CTAs of the unit: those whose ranges hold its first and last pairs, and all between
      const uint64_t c0 = ((unit0 + 1) * grid - 1) / all, c1 = (unit1 * grid - 1) / all;
      uint32_t *cnt = &p.cnt[((size_t)s * hk + kvh) * p.max_blocks + block];
      __threadfence();
      __syncthreads();
      if (t == 0) ticket = atomicAdd(cnt, 1u);
      __syncthreads();
      if (ticket == (uint32_t)(c1 - c0)) {
        __threadfence();
        if (t == 0) *cnt = 0;
        join_parts<HD, MR>(p, w, kvh, block, c0, (uint32_t)(c1 - c0 + 1), unit0, all, grid, reinterpret_cast<float *>(smem));
      }
    }
    at = unit0 + tile1;
  }
}

// ---- more than 32 rows: tcgen05 --------------------------------------------------------------
//
// The same sums for row tiles of 128 on the fifth-generation tensor cores, one CTA an SM. Key tiles of 128
// positions; S = Q K^T and the tile's P V go to TMEM, with K, V and Q (both fp16 parts) in shared memory in the
// 128-byte swizzle and P (both parts) written over S. P V reads V as it lies, hd contiguous (an MN-major B).
//   warps 0-3, 4-7   softmax of every other key tile, a row a thread: maximum and weights
//   warps 8-11       add the tiles' P V to the running output in registers, a row a thread
//   warp 12          issues the MMAs: Q K^T of tile i + 1 before P V of tile i, so that they overlap the softmax
//   warp 13, 14      copy the K and the V tiles by tensor copies, a page or a share of one at a time (p.chunk
//                    positions: the largest power of two up to 128 that divides the page size)
//   warp 15          takes non-finite elements out of V tiles that hold nodes
// Registers: 512 threads at 128; setmaxnreg gives the softmax warps 136, the folding ones 184 and leaves 56 to the
// others (256 * 136 + 128 * 184 + 128 * 56 = 65536, what the block was launched with).
// Calls of at most 32 rows a kv head take row tiles of 32: Q is then small enough for a third K and V tile in flight.
constexpr uint32_t kTcThreads = 512, kTcTile = 128, kTcGrid = 148;

__device__ __forceinline__ uint64_t desc_k(uint32_t saddr) {  // K-major, 128-byte swizzle, 8-row groups of 1024 bytes
  return (uint64_t)((saddr >> 4) & 0x3FFFu) | (uint64_t)1u << 16 | (uint64_t)(1024u >> 4) << 32 | (uint64_t)1u << 46 |
         (uint64_t)2u << 61;
}
__device__ __forceinline__ uint64_t desc_mn(uint32_t saddr, uint32_t block) {
  // MN-major: 64-element blocks of the contiguous dimension `block` bytes apart, 8-row groups of 1024 bytes
  return (uint64_t)((saddr >> 4) & 0x3FFFu) | (uint64_t)(block >> 4) << 16 | (uint64_t)(1024u >> 4) << 32 |
         (uint64_t)1u << 46 | (uint64_t)2u << 61;
}
// kind::f16: fp16 A and B, fp32 sums, M = 128, N = n; b_mn: B is MN-major
__host__ __device__ constexpr uint32_t idesc_f16(uint32_t n, bool b_mn) {
  return (1u << 4) | (b_mn ? 1u << 16 : 0u) | ((n >> 3) << 17) | ((128u >> 4) << 24);
}
// Issued by the one lane that has `leader` set; the whole warp runs the loop around it, so that descriptors stay in
// uniform registers.
__device__ __forceinline__ void tc_mma_ss(uint32_t leader, uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool add) {
  asm volatile(
      "{\n .reg .pred p, q;\n setp.ne.b32 p, %4, 0;\n setp.ne.b32 q, %5, 0;\n"
      " @q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}\n" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"((uint32_t)add), "r"(leader)
      : "memory");
}
__device__ __forceinline__ void tc_mma_ts(uint32_t leader, uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, bool add) {
  asm volatile(
      "{\n .reg .pred p, q;\n setp.ne.b32 p, %4, 0;\n setp.ne.b32 q, %5, 0;\n"
      " @q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}\n" ::"r"(d),
      "r"(a), "l"(b), "r"(idesc), "r"((uint32_t)add), "r"(leader)
      : "memory");
}
__device__ __forceinline__ void tc_commit(uint32_t leader, uint64_t *bar) {
  asm volatile(
      "{\n .reg .pred q;\n setp.ne.b32 q, %1, 0;\n"
      " @q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n}\n" ::"r"(smem_u32(bar)),
      "r"(leader)
      : "memory");
}
__device__ __forceinline__ uint32_t elect_one() {
  uint32_t is;
  asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.u32 %0, 1, 0, p;\n}\n" : "=r"(is));
  return is;
}
// [64 dims] x [chunk positions] of one kv head of one page; coordinates outside the planes read zeros
__device__ __forceinline__ void tma_load(void *dst, const CUtensorMap *map, uint32_t dim, uint32_t row, uint32_t head,
                                         uint32_t page, uint64_t *bar) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], "
      "[%6];" ::"r"(smem_u32(dst)),
      "l"(map), "r"(dim), "r"(row), "r"(head), "r"(page), "r"(smem_u32(bar))
      : "memory");
}
__device__ __forceinline__ void tc_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_ld32(uint32_t at, uint32_t *r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,"
      "%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
        "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
        "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(at));
}
__device__ __forceinline__ void tc_ld16(uint32_t at, uint32_t (&r)[16]) {  // and wait for it
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];\n"
      "tcgen05.wait::ld.sync.aligned;"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(at)
      : "memory");
}
// Wait for the loads; the words pass through, so that nothing that uses them is moved before the wait.
__device__ __forceinline__ void tc_ld_wait(uint32_t *r) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]),
                 "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13])
               :
               : "memory");
  asm volatile("" : "+r"(r[14]), "+r"(r[15]), "+r"(r[16]), "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]),
                    "+r"(r[21]), "+r"(r[22]), "+r"(r[23]), "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27])
               :: "memory");
  asm volatile("" : "+r"(r[28]), "+r"(r[29]), "+r"(r[30]), "+r"(r[31]) :: "memory");
}
__device__ __forceinline__ void tc_st16(uint32_t at, const uint32_t *r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15};" ::"r"(r[0]),
      "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]),
      "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(at)
      : "memory");
}
template <int ID, int N>
__device__ __forceinline__ void named_sync() {
  __syncwarp();
  asm volatile("bar.sync %0, %1;" ::"n"(ID), "n"(N) : "memory");
}

// One CTA's run over the (unit, tile) pairs: the part of each unit that lies in it, in order.
struct Segment {
  SeqWork w;
  uint64_t unit0;
  uint32_t s, kvh, block, tile0, tile1;
  __device__ __forceinline__ bool whole() const { return tile0 == 0 && tile1 == w.tiles; }
};
struct Walk {
  uint64_t at, end;
  uint32_t s;
};
template <uint32_t MR, uint32_t KT>
__device__ __forceinline__ bool next_segment(const TreeParams &p, const uint64_t *upto, Walk &k, Segment &g) {
  if (k.at >= k.end) return false;
  while (upto[k.s + 1] <= k.at) k.s++;
  g.s = k.s;
  g.w = seq_work<MR, KT>(p, k.s);
  const uint64_t unit = (k.at - upto[k.s]) / g.w.tiles;
  g.unit0 = upto[k.s] + unit * g.w.tiles;
  g.kvh = (uint32_t)(unit / g.w.blocks), g.block = (uint32_t)(unit % g.w.blocks);
  const uint64_t unit1 = g.unit0 + g.w.tiles;
  g.tile0 = (uint32_t)(k.at - g.unit0), g.tile1 = (uint32_t)((k.end < unit1 ? k.end : unit1) - g.unit0);
  k.at = g.unit0 + g.tile1;
  return true;
}

template <int HD, uint32_t MR, uint32_t NS>
struct TcSmem {
  static constexpr uint32_t kBlock = kTcTile * 128;         // a tile's 64 dims: 16 KB
  static constexpr uint32_t kTileBytes = HD / 64 * kBlock;  // a K or V tile
  static constexpr uint32_t kQBlock = MR * 128, kQBytes = HD / 64 * kQBlock;  // one part of Q
  // With MR below 128 the MMAs read 128 rows all the same: what follows Q, for rows that nobody reads.
  uint8_t q[2][kQBytes];
  uint8_t kt[NS][kTileBytes];
  uint8_t vt[NS][kTileBytes];
  // Words and rows of a tile are read long before the tile that takes their place: fold(i) frees the TMEM of P V of
  // tile i + 2, so no warp is more than a few tiles ahead of it.
  uint32_t valid[8][4];       // positions of a tile that hold a row
  uint32_t odd[8][4];         // its nodes with a non-finite V row
  float mrow[4][MR];          // [tile]: the maximum that a row's weights of this tile are relative to
  float ml[4][2][MR][2];      // [segment][warpgroup]: a row's maximum and sum of weights
  float factor[MR];
  uint64_t upto[kMaxSeqs + 1];
  uint64_t kfull[NS], kempty[NS], vfull[NS], vclean[NS], vempty[NS], sfull[2], pfull[2], ofull[2], ofree[2], lfull[4],
      qfull, drain;
  uint32_t tmem;
};

template <int HD, uint32_t MR, uint32_t NS>
__global__ void __launch_bounds__(kTcThreads, 1)
    k_attn_tree_tc(TreeParams p, const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap) {
  using Smem = TcSmem<HD, MR, NS>;
  extern __shared__ __align__(16) uint8_t raw[];
  Smem &sm = *reinterpret_cast<Smem *>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~(uintptr_t)1023);
  constexpr uint32_t BL = Smem::kBlock;
  const uint32_t t = threadIdx.x, lane = t & 31, warp = t >> 5;
  pdl_trigger();
  if (t == 0) {
    for (uint32_t i = 0; i < NS; i++) {
      mbar_init(&sm.kfull[i], 1);
      mbar_init(&sm.vfull[i], 1);
      mbar_init(&sm.vclean[i], 32);
      mbar_init(&sm.kempty[i], 1);
      mbar_init(&sm.vempty[i], 1);
    }
    for (int i = 0; i < 2; i++) {
      mbar_init(&sm.sfull[i], 1);
      mbar_init(&sm.pfull[i], 4);
      mbar_init(&sm.ofull[i], 1);
      mbar_init(&sm.ofree[i], 4);
    }
    mbar_init(&sm.qfull, 8);
    for (int i = 0; i < 4; i++) mbar_init(&sm.lfull[i], 8);
    mbar_init(&sm.drain, 1);
    fence_mbar_init();
  }
  if (warp == 12) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&sm.tmem)), "r"(512));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  pdl_wait();
  pairs_before<MR, kTcTile, kTcThreads>(p, sm.upto);
  tc_before();
  __syncthreads();
  tc_after();
  const uint32_t tmem = sm.tmem;
  const uint64_t all = sm.upto[p.c.n_seq], cta = blockIdx.x, grid = gridDim.x < all ? gridDim.x : all;
  Walk walk;
  walk.at = cta < grid ? cta * all / grid : 0;
  walk.end = cta < grid ? (cta + 1) * all / grid : 0;
  walk.s = 0;
  const uint64_t begin = walk.at;
  Segment g;
  bool ok = true;
  // after a wait has run out a role goes on without waiting or copying, so that the barriers among its own threads
  // still meet; the error word tells the host
  auto wait = [&](uint64_t *bar, uint32_t parity) {
    if (ok && !mbar_wait(bar, parity & 1u, p.wait_ns)) {
      ok = false;
      atomicExch(p.err, 1u);
    }
  };
  // which of the 64 positions from node `base32` (negative: committed) on a row of node `nd` may see
  auto seen = [&](uint32_t base32, bool live, uint32_t nd, uint32_t first) -> uint64_t {
    const int32_t base = (int32_t)base32;
    const uint64_t past = low_bits(-(int64_t)base);
    if (!live) return past;
    if (!p.mask) return low_bits((int64_t)nd + 1 - base);
    return past | (window(p.mask + (size_t)(first + nd) * p.words, p.words, base) & ~past);
  };

  if (warp >= 12) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 56;");
    if (warp == 15) {
      // ---- cleaner: V tiles on their way to the MMAs, the rows of those that hold nodes ----
      // (It hands every tile over: a barrier that it watched for some phases only could be two phases on.)
      // A non-finite V row may only reach the rows that see its node, and a weight of 0 does not keep it out of a
      // product: such elements (those of stale rows behind the last node too) become 0 here, and the folding warps
      // add them to the rows that see them.
      constexpr uint32_t CH = HD / 8;
      uint32_t i = 0;
      while (next_segment<MR, kTcTile>(p, sm.upto, walk, g))
        for (uint32_t tile = g.tile0; tile < g.tile1; tile++, i++) {
          const uint32_t sl = i % NS;
          wait(&sm.vfull[sl], i / NS);
          if ((tile + 1) * kTcTile <= g.w.len) {
            mbar_arrive(&sm.vclean[sl]);
            continue;
          }
          uint32_t any[4] = {0, 0, 0, 0};
          // a lane has rows lane, lane + 32, ..: its rows of a word are one bit each
#pragma unroll
          for (uint32_t x = 0; x < 4; x++) {
            const uint32_t r = 32 * x + lane;
            bool bad = false;
#pragma unroll 4
            for (uint32_t ch = 0; ch < CH; ch++) {
              uint4 *at = reinterpret_cast<uint4 *>(sm.vt[sl] + (ch / 8) * BL + r * 128 + (((ch % 8) ^ (r & 7)) << 4));
              uint4 v = *at;
              uint32_t *cw = reinterpret_cast<uint32_t *>(&v);
              bool here = false;
#pragma unroll
              for (int y = 0; y < 4; y++) {
                if ((cw[y] & 0x7C00u) == 0x7C00u) cw[y] &= 0xFFFF0000u, here = true;
                if ((cw[y] & 0x7C000000u) == 0x7C000000u) cw[y] &= 0xFFFFu, here = true;
              }
              if (here) *at = v;
              bad |= here;
            }
            any[x] = __ballot_sync(0xffffffffu, bad);
          }
          if (lane < 4) sm.odd[i & 7][lane] = lane == 0 ? any[0] : lane == 1 ? any[1] : lane == 2 ? any[2] : any[3];
          fence_proxy_async();
          mbar_arrive(&sm.vclean[sl]);
        }
    } else if (warp >= 13) {
      // ---- copies: warp 13 the K tiles, 14 the V tiles; a lane a chunk of p.chunk positions, which lie in one page ----
      const bool is_v = warp == 14;
      const CUtensorMap *map = is_v ? &vmap : &kmap;
      uint64_t *full = is_v ? sm.vfull : sm.kfull, *empty = is_v ? sm.vempty : sm.kempty;
      const uint32_t chunks = kTcTile / p.chunk, chunk = p.chunk, P = p.c.page_tokens;
      uint32_t i = 0;  // tiles of the run so far
      while (next_segment<MR, kTcTile>(p, sm.upto, walk, g)) {
        const uint32_t total = g.w.len + g.w.nodes;
        // where the lane's chunk of a tile lies: page (n_pages for a hole, which reads zeros), first row; -1: behind
        // the last position, not copied
        int32_t page, row;
        auto find = [&](uint32_t tile) {
          const uint32_t pos = tile * kTcTile + lane * chunk;
          page = -1, row = 0;
          if (lane < chunks && tile < g.tile1 && pos < total) {
            const uint32_t pg = pos / P;
            uint32_t x = p.c.n_pages;
            if (pg < p.c.max_pages) x = p.c.table ? (uint32_t)p.c.table[(size_t)g.s * p.c.max_pages + pg] : g.s;
            page = (int32_t)min(x, p.c.n_pages);
            row = (int32_t)(pos - pg * P);
          }
        };
        find(g.tile0);
        for (uint32_t tile = g.tile0; tile < g.tile1; tile++, i++) {
          const uint32_t sl = i % NS;
          const int32_t at = page, r = row;
          find(tile + 1);  // the next tile's table entries come while this one is copied
          const uint32_t copied = __ballot_sync(0xffffffffu, at >= 0);
          const uint32_t there = __ballot_sync(0xffffffffu, at >= 0 && at < (int32_t)p.c.n_pages);
          if (i >= NS) wait(&empty[sl], i / NS - 1);
          __syncwarp();
          if (!is_v) {
            if (lane < 4) {  // the word of positions 32 lane .. + 31
              const uint32_t cap = min(total, p.c.max_pages * P), pos = tile * kTcTile + 32 * lane;
              uint32_t bits = 0;
              if (chunk >= 32) {
                bits = (there >> (32 * lane / chunk)) & 1 ? 0xFFFFFFFFu : 0u;
              } else {
                for (uint32_t c = 0; c < 32 / chunk; c++)
                  if ((there >> (32 / chunk * lane + c)) & 1) bits |= ((1u << chunk) - 1) << (c * chunk);
              }
              sm.valid[i & 7][lane] = bits & (uint32_t)low_bits((int64_t)cap - pos);
            }
            __syncwarp();
          }
          if (ok) {
            uint8_t *dst = (is_v ? sm.vt : sm.kt)[sl] + lane * chunk * 128;
            if (lane == 0) mbar_expect_tx(&full[sl], __popc(copied) * chunk * HD * 2);
            __syncwarp();
            if (at >= 0) {
#pragma unroll
              for (uint32_t b = 0; b < HD / 64; b++) tma_load(dst + b * BL, map, 64 * b, r, g.kvh, at, &full[sl]);
            }
          }
          __syncwarp();
        }
      }
      // the last copies land before the block ends, whatever became of the others
      ok = true;
      for (uint32_t n = i < NS ? 0 : i - NS; n < i; n++) wait(&full[n % NS], n / NS);
    } else {
      // ---- MMA issue ----
      const uint32_t leader = elect_one();
      const uint64_t qd = desc_k(smem_u32(sm.q[0])), kd = desc_k(smem_u32(sm.kt[0])), vd = desc_mn(smem_u32(sm.vt[0]), BL);
      constexpr uint64_t kTileStep = Smem::kTileBytes >> 4, kQStep = Smem::kQBytes >> 4;  // in 16 bytes
      uint32_t i = 0, seg = 0;
      auto scores = [&](uint32_t n) {  // S = Q K^T of tile n: both parts of Q
        wait(&sm.kfull[n % NS], n / NS);
        tc_after();
        const uint64_t kb = kd + (n % NS) * kTileStep;
        const uint32_t d = tmem + 128 * (n & 1);
        if (ok) {
#pragma unroll
          for (uint32_t k = 0; k < HD / 16; k++) {
            const uint64_t qo = ((k / 4) * Smem::kQBlock + (k % 4) * 32) >> 4, ko = ((k / 4) * BL + (k % 4) * 32) >> 4;
            tc_mma_ss(leader, d, qd + qo, kb + ko, idesc_f16(kTcTile, false), k > 0);
            tc_mma_ss(leader, d, qd + kQStep + qo, kb + ko, idesc_f16(kTcTile, false), true);
          }
          tc_commit(leader, &sm.sfull[n & 1]);
          tc_commit(leader, &sm.kempty[n % NS]);
        }
        __syncwarp();
      };
      while (next_segment<MR, kTcTile>(p, sm.upto, walk, g)) {
        wait(&sm.qfull, seg++);
        scores(i);
        for (uint32_t tile = g.tile0; tile < g.tile1; tile++, i++) {
          const uint32_t sl = i % NS;
          if (tile + 1 < g.tile1) scores(i + 1);
          if (i >= 2) wait(&sm.ofree[i & 1], (i >> 1) - 1);
          wait(&sm.pfull[i & 1], i >> 1);
          wait(&sm.vclean[sl], i / NS);
          tc_after();
          const uint64_t vb = vd + sl * kTileStep;
          const uint32_t a = tmem + 128 * (i & 1), d = tmem + 256 + 128 * (i & 1);
          if (ok) {  // this tile's P V, from zero: the sum over tiles is made in registers, where it is rounded
#pragma unroll
            for (uint32_t k = 0; k < kTcTile / 16; k++) {
              const uint32_t at = a + 16 * k;  // 8 words of parts, 8 of remainders
              tc_mma_ts(leader, d, at, vb + k * (2048 >> 4), idesc_f16(HD, true), k > 0);
              tc_mma_ts(leader, d, at + 8, vb + k * (2048 >> 4), idesc_f16(HD, true), true);
            }
            tc_commit(leader, &sm.ofull[i & 1]);
            tc_commit(leader, &sm.vempty[sl]);
          }
          __syncwarp();
        }
      }
      // the MMAs in flight end before TMEM is given back
      tc_commit(leader, &sm.drain);
      ok = true;
      wait(&sm.drain, 0);
      __syncwarp();
    }
  } else if (warp >= 8) {
    // ---- fold: P V of the tiles, in order, into a row's running output; a thread a row ----
    asm volatile("setmaxnreg.inc.sync.aligned.u32 184;");
    const uint32_t r = t & 127, lanes = (warp & 3) * 32 << 16;
    uint32_t i = 0, seg = 0;
    while (next_segment<MR, kTcTile>(p, sm.upto, walk, g)) {
      const uint32_t rows = min(MR, g.w.nodes * p.g - g.block * MR);
      const bool work = (warp & 3) * 32 < rows;  // a warp whose rows are all past the last one keeps step only
      const uint32_t rr = g.block * MR + r, nd = rr / p.g;
      const bool live = r < rows;
      float o[HD], M = -INFINITY;
#pragma unroll
      for (int d = 0; d < HD; d++) o[d] = 0.0f;
      for (uint32_t tile = g.tile0; tile < g.tile1; tile++, i++) {
        wait(&sm.ofull[i & 1], i >> 1);
        __syncwarp();
        tc_after();
        if (work) {
          // the weights of even and odd tiles are relative to maxima of their own
          const float mt = sm.mrow[i & 3][r], mn = fmaxf(M, mt);
          const float a = M == mn ? 1.0f : ex2(M - mn), b = mt == mn ? 1.0f : ex2(mt - mn);
          M = mn;
          const uint32_t oa = tmem + lanes + 256 + 128 * (i & 1);
          const bool plain = __all_sync(0xffffffffu, a == 1.0f && b == 1.0f);
#pragma unroll
          for (int c = 0; c < HD / 16; c++) {
            uint32_t v[16];
            tc_ld16(oa + 16 * c, v);
            if (plain) {
#pragma unroll
              for (int d = 0; d < 16; d++) o[16 * c + d] += __uint_as_float(v[d]);
            } else {
#pragma unroll
              for (int d = 0; d < 16; d++) o[16 * c + d] = fmaf(o[16 * c + d], a, __uint_as_float(v[d]) * b);
            }
          }
        }
        tc_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&sm.ofree[i & 1]);
        if (work && (tile + 1) * kTcTile > g.w.len) {
          // non-finite V elements of nodes that this row sees
#pragma unroll 1
          for (int x = 0; x < 4; x++) {
            uint32_t left = sm.odd[i & 7][x] & sm.valid[i & 7][x];
            if (left) left &= (uint32_t)(seen(tile * kTcTile + 32 * x - g.w.len, live, nd, g.w.first));
#pragma unroll 1
            for (; left; left &= left - 1) {
              const int64_t at_row = kv_row(p.c, g.s, tile * kTcTile + 32 * x + __ffs(left) - 1);
              const __half2 *vr = reinterpret_cast<const __half2 *>(p.c.v + (size_t)g.kvh * p.c.head_stride + at_row);
#pragma unroll
              for (int d = 0; d < HD / 2; d++) {
                const float2 f = __half22float2(vr[d]);
                if (!isfinite(f.x)) o[2 * d] += f.x;
                if (!isfinite(f.y)) o[2 * d + 1] += f.y;
              }
            }
          }
          __syncwarp();
        }
      }
      wait(&sm.lfull[seg & 3], seg >> 2);  // the softmax warps may be two segments ahead, never four
      __syncwarp();
      const bool whole = g.whole();
      if (live) {
        float L = 0.0f;
#pragma unroll
        for (int y = 0; y < 2; y++) {
          const float my = sm.ml[seg & 3][y][r][0];
          if (my != -INFINITY) L = fmaf(sm.ml[seg & 3][y][r][1], my == M ? 1.0f : ex2(my - M), L);
        }
        const uint64_t slot = 2 * cta + (begin >= g.unit0 ? 0 : 1);
        const float scale = whole ? (L != 0.0f ? 1.0f / L : 0.0f) : 1.0f;  // a row that sees nothing gets zeros
        // whole units go to their rows of out; parts lie [hd / 4][row] float4
        float *dst = whole ? p.out + ((size_t)(g.w.first + nd) * p.h + g.kvh * p.g + rr % p.g) * HD
                           : p.part_o + (slot * (HD / 4) * MR + r) * 4;
        const uint32_t step = whole ? 4 : 4 * MR;
#pragma unroll
        for (int d = 0; d < HD; d += 4)
          *reinterpret_cast<float4 *>(dst + (size_t)(d / 4) * step) =
              make_float4(o[d] * scale, o[d + 1] * scale, o[d + 2] * scale, o[d + 3] * scale);
        if (!whole) {
          p.part_ml[(slot * MR + r) * 2] = M;
          p.part_ml[(slot * MR + r) * 2 + 1] = L;
        }
      }
      if (g.tile0 == 0 && r == 0) {
        // for the joining kernel: how many CTAs hold parts of the unit (0: it is whole), and the first one's slot
        const uint64_t c0 = ((g.unit0 + 1) * grid - 1) / all, c1 = ((g.unit0 + g.w.tiles) * grid - 1) / all;
        uint32_t *u = p.units + 2 * (((size_t)g.s * p.c.hk + g.kvh) * p.max_blocks + g.block);
        u[0] = whole ? 0 : (uint32_t)(c1 - c0 + 1);
        u[1] = (uint32_t)(2 * c0 + (c0 * all / grid < g.unit0 ? 1 : 0));
      }
      seg++;
    }
  } else {
    // ---- softmax: warpgroup wg has every other tile of the run, a thread a row ----
    asm volatile("setmaxnreg.inc.sync.aligned.u32 136;");
    const uint32_t wg = warp >> 2, r = t & 127;
    const uint32_t sa = tmem + ((warp & 3) * 32 << 16) + 128 * wg;
    uint32_t i = 0, seg = 0;
    while (next_segment<MR, kTcTile>(p, sm.upto, walk, g)) {
      const uint32_t rows = min(MR, g.w.nodes * p.g - g.block * MR);
      // Q into shared memory, a power of two and two fp16 parts a row; the last segment's products are done
      {
        constexpr uint32_t LR = HD / 4, RW = 32 / LR, WR = MR / 8;  // lanes of a row, rows of an access, rows of a warp
        constexpr uint32_t UN = WR / RW < 4 ? WR / RW : 4;
        const uint32_t d4 = lane % LR;
        for (uint32_t b0 = 0; b0 < WR; b0 += UN * RW) {
          float4 f[UN];
#pragma unroll
          for (uint32_t u = 0; u < UN; u++) {
            const uint32_t rl = warp * WR + b0 + u * RW + lane / LR, rr = g.block * MR + rl;
            f[u] = rl < rows ? *reinterpret_cast<const float4 *>(
                                   p.q + ((size_t)(g.w.first + rr / p.g) * p.h + g.kvh * p.g + rr % p.g) * HD + 4 * d4)
                             : make_float4(0.f, 0.f, 0.f, 0.f);
          }
#pragma unroll
          for (uint32_t u = 0; u < UN; u++) {
            const uint32_t rl = warp * WR + b0 + u * RW + lane / LR;
            float top = fmaxf(fmaxf(fabsf(f[u].x), fabsf(f[u].y)), fmaxf(fabsf(f[u].z), fabsf(f[u].w)));
#pragma unroll
            for (uint32_t o = LR / 2; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
            float down, up;
            row_scale(top, down, up);
            uint2 hi, lo;
            split_f16(f[u].x * down, f[u].y * down, hi.x, lo.x);
            split_f16(f[u].z * down, f[u].w * down, hi.y, lo.y);
            const uint32_t at = (d4 / 16) * Smem::kQBlock + rl * 128 + (((d4 % 16) / 2 ^ (rl & 7)) << 4) + (d4 & 1) * 8;
            *reinterpret_cast<uint2 *>(sm.q[0] + at) = hi;
            *reinterpret_cast<uint2 *>(sm.q[1] + at) = lo;
            if (d4 == 0) sm.factor[rl] = p.scale * up;
          }
        }
        fence_proxy_async();
        __syncwarp();
        if (lane == 0) mbar_arrive(&sm.qfull);
        named_sync<1, 256>();
      }
      const bool work = (warp & 3) * 32 < rows, live = r < rows;
      const float factor = work ? sm.factor[r] : 0.0f;
      const uint32_t nd = (g.block * MR + r) / p.g;
      float m = -INFINITY, l = 0.0f;
      for (uint32_t tile = g.tile0; tile < g.tile1; tile++, i++) {
        if ((i & 1) != wg) continue;
        wait(&sm.sfull[wg], i >> 1);
        __syncwarp();
        tc_after();
        if (work) {
          // Two passes over the scores in steps of 64, rolled: unrolled over the tile, the code of the three
          // warps that share a scheduler outgrew the instruction cache (4 of 14 stalled warps waited for
          // instructions, and a tile took 4000 cycles).
          const bool drafted = (tile + 1) * kTcTile > g.w.len;
          const uint32_t *ok4 = sm.valid[i & 7];
          const bool masked = drafted || (ok4[0] & ok4[1] & ok4[2] & ok4[3]) != ~0u;
          float t4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll 1
          for (uint32_t h = 0; h < 128; h += 64) {
            uint32_t v[64];
            tc_ld32(sa + h, v);
            tc_ld32(sa + h + 32, v + 32);
            tc_ld_wait(v);
            tc_ld_wait(v + 32);
            if (masked) {  // unseen positions become -inf, for the second pass too
              uint64_t see = (uint64_t)ok4[h / 32] | (uint64_t)ok4[h / 32 + 1] << 32;
              if (drafted) see &= seen(tile * kTcTile + h - g.w.len, live, nd, g.w.first);
              const uint32_t b0 = (uint32_t)see, b1 = (uint32_t)(see >> 32);
#pragma unroll
              for (int e = 0; e < 64; e++)
                if (!(((e < 32 ? b0 : b1) >> (e & 31)) & 1)) v[e] = 0xFF800000u;
#pragma unroll
              for (int e = 0; e < 64; e += 16) tc_st16(sa + h + e, v + e);
            }
#pragma unroll
            for (int e = 0; e < 64; e += 8)
#pragma unroll
              for (int u = 0; u < 4; u++)
                t4[u] = fmaxf(t4[u], fmaxf(__uint_as_float(v[e + 2 * u]), __uint_as_float(v[e + 2 * u + 1])));
          }
          if (masked) asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
          const float mn = fmaxf(m, fmaxf(fmaxf(t4[0], t4[1]), fmaxf(t4[2], t4[3])) * factor);
          const float corr = m == mn ? 1.0f : ex2(m - mn);
          m = mn;
          sm.mrow[i & 3][r] = mn;
          __syncwarp();
          const float sub = mn == -INFINITY ? 0.0f : mn - kPShift;
          float part[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 1
          for (uint32_t h = 0; h < 128; h += 64) {  // the weights, over the scores
            uint32_t v[64];
            tc_ld32(sa + h, v);
            tc_ld32(sa + h + 32, v + 32);
            tc_ld_wait(v);
            tc_ld_wait(v + 32);
#pragma unroll
            for (int c = 0; c < 64; c += 16) {
              uint32_t w[16];  // 8 words of parts, 8 of remainders
#pragma unroll
              for (int e = 0; e < 16; e += 2) {
                const float p0 = ex2(fmaf(__uint_as_float(v[c + e]), factor, -sub));
                const float p1 = ex2(fmaf(__uint_as_float(v[c + e + 1]), factor, -sub));
                part[(e / 2) & 3] += p0 + p1;
                split_f16(p0, p1, w[e / 2], w[8 + e / 2]);
              }
              tc_st16(sa + h + c, w);
            }
          }
          l = l * corr + ((part[0] + part[1]) + (part[2] + part[3]));
          asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
        }
        tc_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&sm.pfull[wg]);
      }
      if (work) {
        sm.ml[seg & 3][wg][r][0] = m;
        sm.ml[seg & 3][wg][r][1] = l;
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&sm.lfull[seg & 3]);
      named_sync<1, 256>();  // every score of the segment has been read: Q may be written again
      seg++;
    }
  }
  tc_before();
  __syncthreads();
  if (warp == 12) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512));
}

// Join the parts of the units that several CTAs shared: CTA (unit, 8 rows), a thread 4 dims of a row.
constexpr uint32_t kJoinRows = 8;
template <int HD, uint32_t MR>
__global__ void __launch_bounds__(kJoinRows * HD / 4) k_attn_tree_join(TreeParams p) {
  pdl_trigger();
  pdl_wait();
  __shared__ float ws[kJoinRows][kTcGrid];
  __shared__ float inv[kJoinRows];
  const uint32_t unit = blockIdx.x, block = unit % p.max_blocks, kvh = unit / p.max_blocks % p.c.hk;
  const uint32_t s = unit / p.max_blocks / p.c.hk, row0 = blockIdx.y * kJoinRows, t = threadIdx.x;
  const SeqWork w = seq_work<MR, kTcTile>(p, s);
  if (block >= w.blocks) return;
  const uint32_t rows = min(MR, w.nodes * p.g - block * MR);
  const uint32_t parts = min(p.units[2 * unit], kTcGrid), first = p.units[2 * unit + 1];
  if (parts == 0 || row0 >= rows) return;
  auto slot = [&](uint32_t q) -> size_t { return q == 0 ? first : (first & ~1u) + 2 * q; };
  const uint32_t n = min(kJoinRows, rows - row0), warps = kJoinRows * HD / 128, lane = t & 31;
  for (uint32_t r = t >> 5; r < n; r += warps) {
    float M = -INFINITY;
    for (uint32_t q = lane; q < parts; q += 32) {
      ws[r][q] = p.part_ml[(slot(q) * MR + row0 + r) * 2];
      M = fmaxf(M, ws[r][q]);
    }
    M = warp_max(M);
    float L = 0.0f;
    for (uint32_t q = lane; q < parts; q += 32) {
      const float e = ws[r][q] == -INFINITY ? 0.0f : ex2(ws[r][q] - M);
      L = fmaf(p.part_ml[(slot(q) * MR + row0 + r) * 2 + 1], e, L);
      ws[r][q] = e;
    }
    L = warp_sum(L);
    if (lane == 0) inv[r] = L != 0.0f ? 1.0f / L : 0.0f;
  }
  __syncthreads();
  const uint32_t r = t % kJoinRows, d4 = t / kJoinRows;
  if (r >= n) return;
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  for (uint32_t q0 = 0; q0 < parts; q0 += 8) {
    float4 f[8];
#pragma unroll
    for (int u = 0; u < 8; u++)
      if (q0 + u < parts)
        f[u] = *reinterpret_cast<const float4 *>(p.part_o + ((slot(q0 + u) * (HD / 4) + d4) * MR + row0 + r) * 4);
#pragma unroll
    for (int u = 0; u < 8; u++)
      if (q0 + u < parts) {
        const float y = ws[r][q0 + u];
        acc.x = fmaf(f[u].x, y, acc.x), acc.y = fmaf(f[u].y, y, acc.y);
        acc.z = fmaf(f[u].z, y, acc.z), acc.w = fmaf(f[u].w, y, acc.w);
      }
  }
  const uint32_t rr = block * MR + row0 + r;
  const float y = inv[r];
  *reinterpret_cast<float4 *>(p.out + ((size_t)(w.first + rr / p.g) * p.h + kvh * p.g + rr % p.g) * HD + 4 * d4) =
      make_float4(acc.x * y, acc.y * y, acc.z * y, acc.w * y);
}

// Tensor map of a layer's plane: [page][kv head][position][64 dims of hd], boxes of `chunk` positions, 128-byte swizzle.
bool plane_map(const TreeParams &p, const __half *plane, CUtensorMap *map) {
  const auto encode = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(b200_tensor_map_encoder());
  if (!encode) return false;
  const cuuint64_t dims[4] = {p.c.hd, p.c.page_tokens, p.c.hk, p.c.n_pages};
  const cuuint64_t row = p.c.hd * 2ull;  // a stride along a dimension of one is never used
  const cuuint64_t strides[3] = {row, p.c.hk > 1 ? p.c.head_stride * 2 : row, p.c.n_pages > 1 ? p.c.page_stride * 2 : row};
  const cuuint32_t box[4] = {64, p.chunk, 1, 1}, estr[4] = {1, 1, 1, 1};
  return encode(map, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4, const_cast<__half *>(plane), dims, strides, box, estr,
                CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int HD, uint32_t MR, uint32_t NS>
pai_status_t launch_tree_tc(pai_b200_ctx_t *ctx, TreeParams &p, const CUtensorMap &kmap, const CUtensorMap &vmap) {
  constexpr size_t smem = sizeof(TcSmem<HD, MR, NS>) + 1024;
  static SmemOptIn opt;
  pai_status_t st = b200_cuda(opt.ensure(b200_ctx_device(ctx), smem,
                                         [](size_t b) {
                                           return cudaFuncSetAttribute(k_attn_tree_tc<HD, MR, NS>,
                                                                       cudaFuncAttributeMaxDynamicSharedMemorySize, (int)b);
                                         }),
                              "k_attn_tree_tc smem attribute");
  if (st) return st;
  p.max_blocks = (p.max_nodes * p.g + MR - 1) / MR;
  const uint64_t units = (uint64_t)p.c.n_seq * p.c.hk * p.max_blocks;
  if (units > 0x7FFFFFFu) return b200_fail(PAI_ERR_UNSUPPORTED, "attn_tree: %llu row tiles", (unsigned long long)units);
  const uint64_t pairs = units * (((uint64_t)p.c.max_pages * p.c.page_tokens + p.max_nodes + kTcTile - 1) / kTcTile);
  const uint32_t grid = (uint32_t)std::min<uint64_t>(kTcGrid, pairs);
  float *scratch;
  const uint64_t slots = 2ull * grid;
  st = b200_ctx_scratch(ctx, slots * MR * (HD + 2) + 2 * units, 1, &scratch, &p.cnt);
  if (st) return st;
  p.part_o = scratch;
  p.part_ml = scratch + slots * MR * HD;
  p.units = (uint32_t *)(p.part_ml + slots * MR * 2);
  b200_launch(ctx, k_attn_tree_tc<HD, MR, NS>, dim3(grid), dim3(kTcThreads), smem, p, kmap, vmap);
  // the joining kernel is resident before this one ends, and waits for it
  const int pdl = b200_ctx_pdl(ctx);
  b200_ctx_set_pdl(ctx, 1);
  b200_launch(ctx, k_attn_tree_join<HD, MR>, dim3((uint32_t)units, MR / kJoinRows), dim3(kJoinRows * HD / 4), 0, p);
  b200_ctx_set_pdl(ctx, pdl);
  return b200_launched(ctx, 2, "k_attn_tree_tc");
}

template <int HD, int WM>
pai_status_t launch_tree(pai_b200_ctx_t *ctx, TreeParams &p) {
  constexpr uint32_t MR = 16 * WM, WN = 4 / WM;
  constexpr size_t stages = kStages * sizeof(Stage<HD>), join = WN * MR * (HD + 4 + 2) * sizeof(float);
  constexpr size_t weights = MR * (kGrid + 1) * sizeof(float);  // of the parts of one unit
  constexpr size_t smem = std::max(stages, std::max(join, weights));
  static SmemOptIn opt;
  pai_status_t st = b200_cuda(opt.ensure(b200_ctx_device(ctx), smem,
                                         [](size_t b) {
                                           return cudaFuncSetAttribute(k_attn_tree<HD, WM>,
                                                                       cudaFuncAttributeMaxDynamicSharedMemorySize, (int)b);
                                         }),
                              "k_attn_tree smem attribute");
  if (st) return st;
  p.max_blocks = (p.max_nodes * p.g + MR - 1) / MR;
  const uint64_t units = (uint64_t)p.c.n_seq * p.c.hk * p.max_blocks;
  if (units > 0x7FFFFFFu) return b200_fail(PAI_ERR_UNSUPPORTED, "attn_tree: %llu row tiles", (unsigned long long)units);
  // two CTAs an SM, and no more than there can be pairs
  const uint64_t pairs = units * (((uint64_t)p.c.max_pages * p.c.page_tokens + p.max_nodes + kTile - 1) / kTile);
  const uint32_t grid = (uint32_t)std::min<uint64_t>(kGrid, pairs);
  float *scratch;
  st = b200_ctx_scratch(ctx, 2ull * grid * MR * (HD + 2), (uint32_t)units, &scratch, &p.cnt);
  if (st) return st;
  p.part_o = scratch;
  p.part_ml = scratch + 2ull * grid * MR * HD;
  b200_launch(ctx, k_attn_tree<HD, WM>, dim3(grid), dim3(kThreads), smem, p);
  return b200_launched(ctx, 1, "k_attn_tree");
}

template <int HD>
pai_status_t launch_tree_hd(pai_b200_ctx_t *ctx, TreeParams &p) {
  const uint32_t rows = p.max_nodes * p.g;
  // tensor copies take whole shares of a page, a power of two of at least 8 positions
  p.chunk = 128;
  if (p.c.table)
    while (p.chunk > 8 && p.c.page_tokens % p.chunk) p.chunk /= 2;
  CUtensorMap kmap, vmap;
  if ((!p.c.table || p.c.page_tokens % p.chunk == 0) && plane_map(p, p.c.k, &kmap) && plane_map(p, p.c.v, &vmap))
    return rows <= 32 ? launch_tree_tc<HD, 32, 3>(ctx, p, kmap, vmap) : launch_tree_tc<HD, 128, 2>(ctx, p, kmap, vmap);
  if (rows <= 16) return launch_tree<HD, 1>(ctx, p);
  return launch_tree<HD, 4>(ctx, p);
}

}  // namespace

extern "C" pai_status_t pai_b200_attn_tree_f16kv(pai_b200_ctx_t *ctx, const pai_b200_kv_view_t *kv, uint32_t layer,
                                                 uint64_t h, uint64_t rows, uint32_t max_nodes, const int32_t *lens,
                                                 const int32_t *node_off, const uint64_t *mask, const float *q,
                                                 float *out) {
  TreeParams p{};
  if (!ctx) return b200_fail(PAI_ERR_INVALID_ARG, "attn_tree: NULL context");
  pai_status_t st = kv_nodes_check(kv, "attn_tree", layer, h, rows, max_nodes, lens, node_off, p.c);
  if (st) return st;
  if (!q || !out) return b200_fail(PAI_ERR_INVALID_ARG, "attn_tree: NULL");
  if (((uintptr_t)q | (uintptr_t)out) & 15)
    return b200_fail(PAI_ERR_INVALID_ARG, "attn_tree: q and out must be 16-byte aligned");
  if ((uintptr_t)mask & 7) return b200_fail(PAI_ERR_INVALID_ARG, "attn_tree: the mask must be 8-byte aligned");
  if (kv->head_dim != 64 && kv->head_dim != 128)
    return b200_fail(PAI_ERR_UNSUPPORTED, "attn_tree: head_dim %u (64 or 128)", kv->head_dim);
  p.h = (uint32_t)h, p.g = (uint32_t)h / kv->kv_heads, p.max_nodes = max_nodes, p.words = (max_nodes + 63) / 64;
  p.rows = rows, p.lens = lens, p.off = node_off, p.mask = mask, p.q = q, p.out = out;
  p.err = b200_ctx_errflag(ctx), p.wait_ns = b200_ctx_wait_ns(ctx);
  p.scale = 1.4426950408889634f / sqrtf((float)kv->head_dim);
  const CtxDeviceGuard on(ctx);
  if (on.status()) return on.status();
  return kv->head_dim == 64 ? launch_tree_hd<64>(ctx, p) : launch_tree_hd<128>(ctx, p);
}
