// Attention of drafted nodes over a cache view (pai_b200_attn_tree_f16kv): the choice of kernel, and the form that
// takes any page size.
//
//   attn_tree_few.cuh    at most 32 rows (nodes x query heads of a kv head; 16 with head_dim 64) of a sequence: decoding,
//                        small trees
//   attn_tree_many.cuh   more rows
//   k_attn_tree (here)   where tensor copies cannot fetch the cache: page sizes that no power of two from 8 divides
//                        (a page of 8 n positions is fetched in shares), strides beyond a tensor map's
#include <cudaTypedefs.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>

#include "../b200_internal.h"
#include "attn_tree.cuh"
#include "attn_tree_few.cuh"
#include "attn_tree_many.cuh"
#include "attn_tree_tc.cuh"
#include "b200_device.cuh"
#include "kv_view.cuh"

namespace {

// ---- any page size: mma.sync -----------------------------------------------------------------
//
// Tiles of kTile positions by 16-byte asynchronous copies, row by row, so that a page may end anywhere.
constexpr uint32_t kTile = 64, kThreads = 128;
constexpr uint32_t kGrid = 296;  // two CTAs an SM
constexpr int kStages = 3;

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

// WM warps share a tile's rows (16 each), 4 / WM share its positions. Two CTAs an SM need spills with head_dim 128: 24 bytes of
// stores with 16 rows, 132 with 64.
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
          const float a = f.x * p.scale, b = f.y * p.scale;
          qh[k][x + 2 * e] = __float_as_uint(a);
          ql[k][x + 2 * e] = __float_as_uint(b);
          top = fmaxf(top, fmaxf(fabsf(a), fabsf(b)));
        }
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
      float down;
      row_scale(top, down, factor[x]);
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
        sub[x] = mn == -INFINITY ? 0.0f : shifted(mn);
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
        // a share without a maximum has seen nothing (zeros) or only scores that are not numbers (NaN, which stays)
        const float my = sm[(y * MR + r) * 2], wy = my == -INFINITY ? 0.0f : ex2(my - M);
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

// The tcgen05 kernels: `kern` with `smem` bytes and row tiles of MR, then the joining kernel. RG: the groups of 8 rows
// of the kernel for few rows, 0 for that of many (it also keeps the kernels' shared-memory attributes apart).
template <int HD, uint32_t MR, uint32_t RG>
pai_status_t launch_tc(pai_b200_ctx_t *ctx, TreeParams &p, void (*kern)(TreeParams, CUtensorMap, CUtensorMap),
                       uint32_t threads, size_t smem, const CUtensorMap &kmap, const CUtensorMap &vmap) {
  static SmemOptIn opt;
  pai_status_t st = b200_cuda(opt.ensure(b200_ctx_device(ctx), smem,
                                         [kern](size_t b) {
                                           return cudaFuncSetAttribute((const void *)kern,
                                                                       cudaFuncAttributeMaxDynamicSharedMemorySize, (int)b);
                                         }),
                              "attn_tree smem attribute");
  if (st) return st;
  p.max_blocks = (p.max_nodes * p.g + MR - 1) / MR;
  const uint64_t units = (uint64_t)p.c.n_seq * p.c.hk * p.max_blocks;
  if (units > 0x7FFFFFFu) return b200_fail(PAI_ERR_UNSUPPORTED, "attn_tree: %llu row tiles", (unsigned long long)units);
  const uint64_t pairs = units * (((uint64_t)p.c.max_pages * p.c.page_tokens + p.max_nodes + kTcTile - 1) / kTcTile + kStart);
  if (pairs > 0x7FFFFFFFull)  // numbered in 32 bits
    return b200_fail(PAI_ERR_UNSUPPORTED, "attn_tree: %llu tiles of rows and keys", (unsigned long long)pairs);
  const uint32_t grid = (uint32_t)std::min<uint64_t>(kTcGrid, pairs);
  float *scratch;
  const uint64_t slots = 2ull * grid;
  p.slots = (uint32_t)slots;
  st = b200_ctx_scratch(ctx, slots * MR * (HD + 2) + 2 * units, 1, &scratch, &p.cnt);
  if (st) return st;
  p.part_o = scratch;
  p.part_ml = scratch + slots * MR * HD;
  p.units = (uint32_t *)(p.part_ml + slots * MR * 2);
  b200_launch(ctx, kern, dim3(grid), dim3(threads), smem, p, kmap, vmap);
  // the joining kernel is resident before this one ends, and waits for it
  const int pdl = b200_ctx_pdl(ctx);
  b200_ctx_set_pdl(ctx, 1);
  b200_launch(ctx, k_attn_tree_join<HD, MR, RG != 0>, dim3((uint32_t)units, MR / kJoinRows), dim3(kJoinRows * HD / 4), 0, p);
  b200_ctx_set_pdl(ctx, pdl);
  return b200_launched(ctx, 2, "k_attn_tree");
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
  {
    // 8 sequences at 16384 positions, with the exchanged operands and without: 8 rows 93 and 121 us, 32 rows 109 and 127
    // (at 4096 positions 55 and 51, the lengths are not known here); 8 rows with 16 at compile time 97, 16 rows with 32
    // 106 instead of 99. With head_dim 64 a tile is half the bytes and the same softmax: 16 rows 84 and 108, 32 rows 119
    // and 108 (one sequence at 4096: 24.8 and 20.6).
    constexpr uint32_t kMost = HD == 64 ? 16 : kFewRows;
    if (rows > kMost)
      return launch_tc<HD, kManyRows, 0>(ctx, p, k_attn_tree_many<HD>, kManyThreads, sizeof(ManySmem<HD>) + 1024, kmap, vmap);
    constexpr size_t smem = sizeof(FewSmem<HD>) + 1024;
    if (rows <= 8) return launch_tc<HD, kFewRows, 1>(ctx, p, k_attn_tree_few<HD, 1, 1>, few_threads(1), smem, kmap, vmap);
    if (rows <= 16) return launch_tc<HD, kFewRows, 2>(ctx, p, k_attn_tree_few<HD, 2, 1>, few_threads(1), smem, kmap, vmap);
    if constexpr (kMost > 16)
      return launch_tc<HD, kFewRows, 4>(ctx, p, k_attn_tree_few<HD, 2, 2>, few_threads(2), smem, kmap, vmap);
  }
  // 8 sequences at 16384 positions in pages of 100: 16 rows 126 us in tiles of 16, 253 in one of 64; 20 rows (two tiles)
  // 217 and 255; 64 rows 432 and 279
  if (rows <= 32) return launch_tree<HD, 1>(ctx, p);
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
