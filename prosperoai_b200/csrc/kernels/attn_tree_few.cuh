// Tree attention of at most 32 rows a kv head, 16 with head_dim 64 (decoding, small trees): bound by the cache's bytes.
//
// The operands change places, so that the tensor cores and the softmax do the rows' work and not that of 128 rows:
//   S^T = K Q^T      M = 128 positions, N = 64: the 32 rows' fp16 parts, then their remainders
//   O^T = V^T P^T    M = 128 dims (V as it lies, hd contiguous: an MN-major A), N = 64 likewise, K = 128 positions
// A softmax thread has a position and all rows: the weights of a tile need no exchange as long as no row's maximum
// grows by more than 2^3 (they are relative to a maximum that may be that much too small: fp16 holds 2^15.99, and the
// weights carry 2^12). Only when some row's does, in a sequence's first tiles, are the rows' maxima taken over the
// tile. The sums of weights stay in the threads, one a row and position, until a unit ends.
//   first 4 or 8 warps  softmax; the weights go to shared memory, 128 bytes a position, as an MN-major B
//   next 4              add the tiles' O^T to the running output, a thread a dim, the rows in registers
//   last 4              issue the MMAs (8 + 8 of 48 cycles of shared memory a tile), copy K and V, clean V
// With row tiles as A (attn_tree_many.cuh) 8 sequences of one row x 4 heads at 16384 positions took 134 us: 128 rows'
// MMAs, and one warp of four with a row to work on. RG, the groups of 8 rows that a softmax and a folding thread have, is
// a compile-time value: with 1 for 8 rows that took 101 us, with 4 and three of them idle 125 (these warps wait for
// instructions more than for anything else).
#pragma once
#include <cfloat>

#include "attn_tree_tc.cuh"

namespace {

constexpr uint32_t kFewRows = 32;

template <int HD>
struct FewSmem {
  static constexpr uint32_t kBlock = kTcTile * 128;         // a tile's 64 dims: 16 KB
  static constexpr uint32_t kTileBytes = HD / 64 * kBlock;  // a K or V tile
  static constexpr uint32_t kQBlock = 64 * 128;             // 64 dims of the rows' parts and remainders
  // tiles of K and V in flight, 96 and 64 KB (head_dim 64 with half of that: 8 x one token at 16384 62 us instead of 60)
  static constexpr uint32_t kK = 3 * 128 / HD, kV = 2 * 128 / HD;
  static constexpr uint32_t kWords = HD == 64 ? 16 : 8;
  uint8_t q[HD / 64 * kQBlock];
  uint8_t kt[kK][kTileBytes];
  uint8_t vt[kV][kTileBytes];
  uint8_t pt[2][kTcTile * 128];  // weights: [position][32 rows' parts, 32 rows' remainders]
  // Words of a tile are read long before the tile that takes their place: P V of a tile waits for the tile before the
  // last to be folded, and K of a tile for the scores kK tiles before, so no warp is kK + 3 tiles ahead of another.
  uint32_t valid[kWords][4];  // positions of a tile that hold a row
  uint32_t odd[kWords][4];    // its nodes with a non-finite V row
  uint32_t grew[kWords][2];   // [tile][softmax warpgroup]: whether the weights are relative to new maxima
  float corr[kWords][kFewRows];  // then: 2^(old - new)
  float factor[kFewRows], sub[kFewRows];
  float wmax[2][4][kFewRows];
  float lsum[4][4][kFewRows], msum[4][kFewRows];  // [segment][warp]: sums of weights; maxima
  uint32_t upto[kMaxSeqs + 1];
  Ring ring;
  uint64_t kfull[kK], kempty[kK], vfull[kV], vclean[kV], vempty[kV], sfull[2], pfull[2], ofull[2], ofree[2],
      lfull[4], qfull, drain;
  uint32_t tmem;
};

// Threads of a block: SW warpgroups of softmax, one that folds, four warps for the other roles.
__host__ __device__ constexpr uint32_t few_threads(uint32_t sw) { return 128 * (sw + 2); }

// The largest of the lanes' values, NaN apart.
__device__ __forceinline__ float warp_top(float v) {
  float top;
  asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(top) : "f"(v));
  return top;
}

template <int HD, uint32_t RG, uint32_t SW>
__global__ void __launch_bounds__(few_threads(SW), 1)
    k_attn_tree_few(TreeParams p, const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap) {
  using Smem = FewSmem<HD>;
  extern __shared__ __align__(16) uint8_t raw[];
  Smem &sm = *reinterpret_cast<Smem *>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~(uintptr_t)1023);
  constexpr uint32_t kFewK = Smem::kK, kFewV = Smem::kV, WM = Smem::kWords - 1;
  constexpr uint32_t BL = Smem::kBlock, FOLD = 4 * SW, MMA = FOLD + 4;  // first warps of those roles
  const uint32_t t = threadIdx.x, lane = t & 31, warp = t >> 5;
  pdl_trigger();
  if (t == 0) {
    for (uint32_t i = 0; i < kFewK; i++) {
      mbar_init(&sm.kfull[i], 1);
      mbar_init(&sm.kempty[i], 1);
    }
    for (uint32_t i = 0; i < kFewV; i++) {
      mbar_init(&sm.vfull[i], 1);
      mbar_init(&sm.vclean[i], 1);
      mbar_init(&sm.vempty[i], 1);
    }
    for (int i = 0; i < 2; i++) {
      mbar_init(&sm.sfull[i], 1);
      mbar_init(&sm.pfull[i], 4 * SW);
      mbar_init(&sm.ofull[i], 1);
      mbar_init(&sm.ofree[i], 4);
    }
    for (int i = 0; i < 4; i++) mbar_init(&sm.lfull[i], 4 * SW);
    mbar_init(&sm.qfull, 4 * SW);
    mbar_init(&sm.drain, 1);
    for (uint32_t i = 0; i < kRing; i++) mbar_init(&sm.ring.full[i], 1);
    fence_mbar_init();
  }
  if (warp == MMA) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&sm.tmem)), "r"(256));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  pdl_wait();
  pairs_before32<kFewRows, few_threads(SW)>(p, sm.upto);
  tc_before();
  __syncthreads();
  tc_after();
  const uint32_t tmem = sm.tmem;  // columns 0, 64: S^T of even and odd tiles; 128, 192: O^T
  Segment g;
  Waiter wait{p.wait_ns, p.err};
  uint32_t i = 0, seg = 0;  // tiles and segments of the run so far

  if (warp == MMA + 1) {
    copy_tiles<HD, kFewRows, kFewK, true, WM>(p, &kmap, sm.upto, sm.ring, sm.kt[0], sm.kfull, sm.kempty, sm.valid);
  } else if (warp == MMA + 2) {
    copy_tiles<HD, kFewRows, kFewV, false, WM>(p, &vmap, sm.upto, sm.ring, sm.vt[0], sm.vfull, sm.vempty, nullptr);
  } else if (warp == MMA + 3) {
    clean_tiles<HD, kFewV, 1, WM>(p, sm.ring, 0, sm.vt[0], sm.vfull, sm.vclean, sm.odd);
  } else if (warp == MMA) {
    // ---- MMA issue ----
    const uint32_t leader = elect_one();
    const uint64_t qd = desc_k(smem_u32(sm.q)), kd = desc_k(smem_u32(sm.kt[0]));
    const uint64_t vd = desc_mn(smem_u32(sm.vt[0]), BL), pd = desc_mn(smem_u32(sm.pt[0]), 0);
    constexpr uint64_t kStep = Smem::kTileBytes >> 4, kPStep = (kTcTile * 128) >> 4;  // in 16 bytes
    auto scores = [&](uint32_t n) {  // S^T of tile n
      wait(&sm.kfull[n % kFewK], n / kFewK);
      tc_after();
      const uint64_t kb = kd + (n % kFewK) * kStep;
      if (wait.ok) {
#pragma unroll
        for (uint32_t k = 0; k < HD / 16; k++)
          tc_mma_ss(leader, tmem + 64 * (n & 1), kb + (((k / 4) * BL + (k % 4) * 32) >> 4),
                    qd + (((k / 4) * Smem::kQBlock + (k % 4) * 32) >> 4), idesc_f16(64, false), k > 0);
        tc_commit(leader, &sm.sfull[n & 1]);
        tc_commit(leader, &sm.kempty[n % kFewK]);
      }
      __syncwarp();
    };
    for (; next_segment(sm.ring, seg, wait, g); seg++) {
      wait(&sm.qfull, seg);
      scores(i);
      for (uint32_t tile = g.tile0; tile < g.tile1; tile++, i++) {
        if (tile + 1 < g.tile1) scores(i + 1);
        if (i >= 2) wait(&sm.ofree[i & 1], (i >> 1) - 1);
        wait(&sm.vclean[i % kFewV], i / kFewV);
        wait(&sm.pfull[i & 1], i >> 1);
        tc_after();
        const uint64_t vb = vd + (i % kFewV) * kStep, pb = pd + (i & 1) * kPStep;
        if (wait.ok) {  // this tile's O^T, from zero: the sum over tiles is made in registers, where it is rounded
#pragma unroll
          for (uint32_t k = 0; k < kTcTile / 16; k++)
            tc_mma_ss(leader, tmem + 128 + 64 * (i & 1), vb + k * (2048 >> 4), pb + k * (2048 >> 4),
                      idesc_f16(64, true, true), k > 0);
          tc_commit(leader, &sm.ofull[i & 1]);
          tc_commit(leader, &sm.vempty[i % kFewV]);
        }
        __syncwarp();
      }
    }
    // the MMAs in flight end before TMEM is given back
    tc_commit(leader, &sm.drain);
    wait.ok = true;
    wait(&sm.drain, 0);
    __syncwarp();
  } else if (warp >= FOLD) {
    // ---- fold: a thread a dim (with hd 64 the upper half of the lanes has none) ----
    const uint32_t d = t - 32 * FOLD, lanes = (warp & 3) * 32 << 16;
    const bool live = d < HD;
    constexpr uint32_t FR = 8 * RG * SW;  // rows
    for (; next_segment(sm.ring, seg, wait, g); seg++) {
      const uint32_t rows = min(kFewRows, g.nodes * p.g - g.block * kFewRows);
      float o[FR];
#pragma unroll
      for (uint32_t r = 0; r < FR; r++) o[r] = 0.0f;
      for (uint32_t tile = g.tile0; tile < g.tile1; tile++, i++) {
        wait(&sm.ofull[i & 1], i >> 1);
        __syncwarp();
        tc_after();
        uint32_t w[2 * FR];
#pragma unroll
        for (uint32_t gr = 0; gr < FR / 8; gr++) {
          tc_ld8(tmem + lanes + 128 + 64 * (i & 1) + 8 * gr, w + 16 * gr);
          tc_ld8(tmem + lanes + 160 + 64 * (i & 1) + 8 * gr, w + 16 * gr + 8);
        }
#pragma unroll
        for (uint32_t gr = 0; gr < FR / 8; gr++) {
          uint32_t *v = w + 16 * gr;
          if (sm.grew[i & WM][gr / RG]) {
#pragma unroll
            for (uint32_t e = 0; e < 8; e++) o[8 * gr + e] *= sm.corr[i & WM][8 * gr + e];
          }
          tc_ld_wait8(v);
          tc_ld_wait8(v + 8);
#pragma unroll
          for (uint32_t e = 0; e < 8; e++) o[8 * gr + e] += __uint_as_float(v[e]) + __uint_as_float(v[8 + e]);
        }
        tc_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&sm.ofree[i & 1]);
        if ((tile + 1) * kTcTile > g.len && live) {
          // non-finite V elements of nodes, for the rows that see them
#pragma unroll 1
          for (int x = 0; x < 4; x++)
#pragma unroll 1
            for (uint32_t left = sm.odd[i & WM][x] & sm.valid[i & WM][x]; left; left &= left - 1) {
              const uint32_t pos = tile * kTcTile + 32 * x + __ffs(left) - 1;
              // (no row, where a wait has run out and the words are old ones: then the plane's first)
              const int64_t at_row = max(kv_row(p.c, g.s, pos), (int64_t)0);
              const float f = __half2float(p.c.v[(size_t)g.kvh * p.c.head_stride + at_row + d]);
              if (isfinite(f)) continue;
#pragma unroll
              for (uint32_t r = 0; r < FR; r++)
                if (r < rows && sees_node(p, g.first, (g.block * kFewRows + r) / p.g, pos - g.len))
                  o[r] += f;
            }
        }
        __syncwarp();
      }
      wait(&sm.lfull[seg & 3], seg >> 2);  // the softmax warps may be two segments ahead, never four
      __syncwarp();
      const bool whole = g.whole();
      const size_t slot = g.slot;
#pragma unroll
      for (uint32_t r = 0; r < FR; r++) {
        if (r >= rows) continue;
        const float *ls = &sm.lsum[seg & 3][0][r];
        const float L = (ls[0] + ls[kFewRows]) + (ls[2 * kFewRows] + ls[3 * kFewRows]);
        const uint32_t rr = g.block * kFewRows + r;
        if (whole) {  // a row that sees nothing gets zeros
          if (live)
            p.out[((size_t)(g.first + rr / p.g) * p.h + g.kvh * p.g + rr % p.g) * HD + d] = L != 0.0f ? o[r] * (1.0f / L) : 0.0f;
        } else {
          if (live) p.part_o[(slot * kFewRows + r) * HD + d] = o[r];
          if (d == 0) {
            p.part_ml[(slot * kFewRows + r) * 2] = sm.msum[seg & 3][r];
            p.part_ml[(slot * kFewRows + r) * 2 + 1] = L;
          }
        }
      }
      if (g.tile0 == 0 && d == 0) note_unit(p, g);
    }
  } else {
    // ---- softmax: a thread a position and 8 RG rows, from row0 ----
    const uint32_t wg = warp / 4, w4 = warp & 3, row0 = 8 * RG * wg;
    // no maximum yet: below every score; the largest exponent that weights may have
    constexpr float kNone = -FLT_MAX, kFull = 15.5f;
    for (; next_segment<1, 128 * SW>(sm.ring, seg, wait, g); seg++) {
      const uint32_t rows = min(kFewRows, g.nodes * p.g - g.block * kFewRows);
      // every score of the last segment has been read, so its products are done: Q may be written
      put_queries<HD, kFewRows, 4 * SW>(p, g, rows, warp, sm.q, Smem::kQBlock, kFewRows * 128, sm.factor);
      if (t < kFewRows) sm.sub[t] = kNone;
      __syncwarp();
      if (lane == 0) mbar_arrive(&sm.qfull);
      named_sync<1, 128 * SW>();
      float m = -INFINITY;  // of row row0 + lane
      float l[8 * RG];
#pragma unroll
      for (uint32_t r = 0; r < 8 * RG; r++) l[r] = 0.0f;
      for (uint32_t tile = g.tile0; tile < g.tile1; tile++, i++) {
        const uint32_t sa = tmem + (w4 * 32 << 16) + 64 * (i & 1) + row0;
        wait(&sm.sfull[i & 1], i >> 1);
        __syncwarp();
        tc_after();
        const bool there = (sm.valid[i & WM][w4] >> lane) & 1;
        const uint32_t pos = tile * kTcTile + (t & 127);
        const bool is_node = (tile + 1) * kTcTile > g.len && pos >= g.len;
        // scores in powers of two, unseen ones -inf, and the largest exponent relative to the rows' maxima so far
        float s[8 * RG], top = -INFINITY;
        uint32_t w[16 * RG];
#pragma unroll
        for (uint32_t gr = 0; gr < RG; gr++) {
          tc_ld8(sa + 8 * gr, w + 16 * gr);
          tc_ld8(sa + 32 + 8 * gr, w + 16 * gr + 8);
        }
#pragma unroll
        for (uint32_t gr = 0; gr < RG; gr++) {
          uint32_t *v = w + 16 * gr;
          tc_ld_wait8(v);
          tc_ld_wait8(v + 8);
#pragma unroll
          for (uint32_t e = 0; e < 8; e += 4) {
            const uint32_t r = 8 * gr + e;
            const float4 f = *reinterpret_cast<const float4 *>(&sm.factor[row0 + r]);
            const float4 u = *reinterpret_cast<const float4 *>(&sm.sub[row0 + r]);
            s[r] = there ? (__uint_as_float(v[e]) + __uint_as_float(v[8 + e])) * f.x : -INFINITY;
            s[r + 1] = there ? (__uint_as_float(v[e + 1]) + __uint_as_float(v[9 + e])) * f.y : -INFINITY;
            s[r + 2] = there ? (__uint_as_float(v[e + 2]) + __uint_as_float(v[10 + e])) * f.z : -INFINITY;
            s[r + 3] = there ? (__uint_as_float(v[e + 3]) + __uint_as_float(v[11 + e])) * f.w : -INFINITY;
            if (is_node) {  // for the rows that see it
#pragma unroll
              for (uint32_t x = r; x < r + 4; x++)
                if (row0 + x < rows && !sees_node(p, g.first, (g.block * kFewRows + row0 + x) / p.g, pos - g.len)) s[x] = -INFINITY;
            }
            top = fmaxf(fmaxf(top, fmaxf(s[r] - u.x, s[r + 1] - u.y)), fmaxf(s[r + 2] - u.z, s[r + 3] - u.w));
          }
        }
        __syncwarp();
        uint32_t any;  // of this warpgroup's rows
        asm volatile(
            "{\n .reg .pred p, q;\n setp.ne.u32 q, %1, 0;\n bar.red.or.pred p, %2, 128, q;\n selp.u32 %0, 1, 0, p;\n}\n"
            : "=r"(any)
            : "r"((uint32_t)(top > kFull)), "r"(2 + wg)
            : "memory");
        if (any) {
          float mine = -INFINITY;
#pragma unroll
          for (uint32_t gr = 0; gr < RG; gr++) {
#pragma unroll
            for (uint32_t r = 8 * gr; r < 8 * gr + 8; r++) {
              const float x = warp_top(s[r]);
              if (lane == r) mine = x;
            }
          }
          sm.wmax[wg][w4][lane] = mine;
          group_sync(2 + wg);
          const float(*wm)[kFewRows] = sm.wmax[wg];
          const float mn = fmaxf(fmaxf(fmaxf(m, wm[0][lane]), fmaxf(wm[1][lane], wm[2][lane])), wm[3][lane]);
          const float corr = m == mn ? 1.0f : ex2(m - mn);
          m = mn;
          if (w4 == 0 && lane < 8 * RG) {
            sm.sub[row0 + lane] = mn == -INFINITY ? kNone : shifted(mn);
            sm.corr[i & WM][row0 + lane] = corr;
          }
#pragma unroll
          for (uint32_t gr = 0; gr < RG; gr++) {
#pragma unroll
            for (uint32_t r = 8 * gr; r < 8 * gr + 8; r++) l[r] *= __shfl_sync(0xffffffffu, corr, r);
          }
          group_sync(2 + wg);
        }
        if (w4 == 0 && lane == 0) sm.grew[i & WM][wg] = any;
        // weights, in groups of 8 rows, to the position's 128 bytes (16 of parts and 16 of remainders a group)
        uint8_t *dst = sm.pt[i & 1] + (t & 127) * 128;
#pragma unroll
        for (uint32_t gr = 0; gr < RG; gr++) {
          uint4 hi, lo;
          uint32_t *hw = reinterpret_cast<uint32_t *>(&hi), *lw = reinterpret_cast<uint32_t *>(&lo);
#pragma unroll
          for (uint32_t e = 0; e < 8; e += 2) {
            const uint32_t r = 8 * gr + e;
            const float2 u = *reinterpret_cast<const float2 *>(&sm.sub[row0 + r]);
            const float p0 = ex2(s[r] - u.x), p1 = ex2(s[r + 1] - u.y);
            l[r] += p0;
            l[r + 1] += p1;
            split_f16(p0, p1, hw[e / 2], lw[e / 2]);
          }
          const uint32_t c = row0 / 8 + gr;
          *reinterpret_cast<uint4 *>(dst + ((c ^ (t & 7)) << 4)) = hi;
          *reinterpret_cast<uint4 *>(dst + (((4 + c) ^ (t & 7)) << 4)) = lo;
        }
        fence_proxy_async();
        tc_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&sm.pfull[i & 1]);
      }
      // lane r: the warp's sum of row row0 + r
      float sum = 0.0f;
#pragma unroll
      for (uint32_t r = 0; r < 8 * RG; r++) {
        const float x = warp_sum(l[r]);
        if (lane == r) sum = x;
      }
      if (lane < 8 * RG) {
        sm.lsum[seg & 3][w4][row0 + lane] = sum;
        if (w4 == 0) sm.msum[seg & 3][row0 + lane] = m;
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&sm.lfull[seg & 3]);
      named_sync<1, 128 * SW>();  // the factors and maxima may be written again
    }
  }
  tc_before();
  __syncthreads();
  if (warp == MMA) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(256));
}

}  // namespace
