// Tree attention of more than 32 rows a kv head: row tiles of 128.
//
// S = Q K^T (M = 128 rows, N = 128 positions, both fp16 parts of Q) and the tile's P V go to TMEM; P (both parts) is
// written over S and is the A operand of P V, V, as it lies with hd contiguous, an MN-major B.
//   warps 0-15       softmax, a row a thread: every four of them have 32 of a tile's positions; the row's maximum goes
//                    through shared memory. Then the P V of the tile before, which ran meanwhile, is added to the
//                    running output in registers, 32 dims each.
//   warp 16          issues the MMAs: Q K^T of tile i + 1 before P V of tile i, so that they overlap the softmax
//   warps 17-19      K copies, V copies, cleaning
// Registers: 640 threads at 96; setmaxnreg gives the softmax warps 104 and leaves 56 to the others (512 * 104 + 128 * 56
// = 60416 of 61440, what the block was launched with).
//
// 8 sequences of 64 nodes x 4 heads a kv head at 32768 positions: 533 us (1.03 PFLOP/s with both parts) after a second's
// rest, 642 us in a run of seconds, which the power limit holds at 1335 MHz; the same instructions on a cache of zeros take
// 425 us at 1965 MHz. That is 858 and 835 thousand cycles: the clock is what differs. One tree of 16 at 4096: 22.8 us.
// (64 positions a thread instead of 32, with a second pass over the scores for want of registers: 24.7 there, and 1.04
// times as long for the large case on one GPU.) At 96 registers the compiler spills: 48 bytes of stores, 112 of loads.
#pragma once
#include "attn_tree_tc.cuh"

namespace {

constexpr uint32_t kManyGroups = 4, kManySoft = 128 * kManyGroups, kManyThreads = kManySoft + 128, kManyRows = 128;

template <int HD>
struct ManySmem {
  static constexpr uint32_t kBlock = 128 * 128;             // 128 rows of 64 dims: 16 KB
  static constexpr uint32_t kTileBytes = HD / 64 * kBlock;  // a K or V tile, or one part of Q
  uint8_t q[2][kTileBytes];
  static constexpr uint32_t kSlots = 2 * 128 / HD;          // tiles of K and of V in flight, 64 KB each
  uint8_t kt[kSlots][kTileBytes];
  uint8_t vt[kSlots][kTileBytes];
  uint32_t valid[8][4];          // positions of a tile that hold a row; a tile's words are read long before 8 tiles on
  uint32_t odd[8][4];            // its nodes with a non-finite V row
  float factor[kManyRows];
  float top[2][kManyRows][kManyGroups];  // [tile parity]: maxima of a row's quarters
  float ml[kManyGroups][kManyRows];
  uint32_t upto[kMaxSeqs + 1];
  Ring ring;
  uint64_t kfull[kSlots], kempty[kSlots], vfull[kSlots], vclean[kSlots], vempty[kSlots], sfull[2], pfull[2], ofull[2], qfull, drain;
  uint32_t tmem;
};

template <int HD>
__global__ void __launch_bounds__(kManyThreads, 1)
    k_attn_tree_many(TreeParams p, const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap) {
  using Smem = ManySmem<HD>;
  extern __shared__ __align__(16) uint8_t raw[];
  Smem &sm = *reinterpret_cast<Smem *>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~(uintptr_t)1023);
  constexpr uint32_t kSlots = Smem::kSlots, BL = Smem::kBlock, MMA = kManySoft / 32;  // first warp behind the softmax
  const uint32_t t = threadIdx.x, lane = t & 31, warp = t >> 5;
  pdl_trigger();
  if (t == 0) {
    for (uint32_t i = 0; i < kSlots; i++) {
      mbar_init(&sm.kfull[i], 1);
      mbar_init(&sm.vfull[i], 1);
      mbar_init(&sm.vclean[i], 1);
      mbar_init(&sm.kempty[i], 1);
      mbar_init(&sm.vempty[i], 1);
    }
    for (int i = 0; i < 2; i++) {
      mbar_init(&sm.sfull[i], 1);
      mbar_init(&sm.pfull[i], MMA);
      mbar_init(&sm.ofull[i], 1);
    }
    mbar_init(&sm.qfull, MMA);
    mbar_init(&sm.drain, 1);
    for (uint32_t i = 0; i < kRing; i++) mbar_init(&sm.ring.full[i], 1);
    fence_mbar_init();
  }
  if (warp == MMA) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&sm.tmem)), "r"(512));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  pdl_wait();
  pairs_before32<kManyRows, kManyThreads>(p, sm.upto);
  tc_before();
  __syncthreads();
  tc_after();
  const uint32_t tmem = sm.tmem;
  Segment g;
  Waiter wait{p.wait_ns, p.err};

  if (warp >= MMA) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 56;");
    if (warp == MMA + 1) {
      copy_tiles<HD, kManyRows, kSlots, true, 7>(p, &kmap, sm.upto, sm.ring, sm.kt[0], sm.kfull, sm.kempty, sm.valid);
    } else if (warp == MMA + 2) {
      copy_tiles<HD, kManyRows, kSlots, false, 7>(p, &vmap, sm.upto, sm.ring, sm.vt[0], sm.vfull, sm.vempty, nullptr);
    } else if (warp == MMA + 3) {
      clean_tiles<HD, kSlots, 1, 7>(p, sm.ring, 0, sm.vt[0], sm.vfull, sm.vclean, sm.odd);
    } else {
      // ---- MMA issue ----
      const uint32_t leader = elect_one();
      const uint64_t qd = desc_k(smem_u32(sm.q[0])), kd = desc_k(smem_u32(sm.kt[0])), vd = desc_mn(smem_u32(sm.vt[0]), BL);
      constexpr uint64_t kPart = Smem::kTileBytes >> 4;  // from one part of Q, or one tile, to the next, in 16 bytes
      uint32_t i = 0, seg = 0;
      auto scores = [&](uint32_t n) {  // S = Q K^T of tile n: both parts of Q
        wait(&sm.kfull[n % kSlots], n / kSlots);
        tc_after();
        const uint64_t kb = kd + (n % kSlots) * kPart;
        const uint32_t d = tmem + 128 * (n & 1);
        if (wait.ok) {
#pragma unroll
          for (uint32_t k = 0; k < HD / 16; k++) {
            const uint64_t off = ((k / 4) * BL + (k % 4) * 32) >> 4;
            tc_mma_ss(leader, d, qd + off, kb + off, idesc_f16(kTcTile, false), k > 0);
            tc_mma_ss(leader, d, qd + kPart + off, kb + off, idesc_f16(kTcTile, false), true);
          }
          tc_commit(leader, &sm.sfull[n & 1]);
          tc_commit(leader, &sm.kempty[n % kSlots]);
        }
        __syncwarp();
      };
      for (; next_segment(sm.ring, seg, wait, g); seg++) {
        wait(&sm.qfull, seg);
        scores(i);
        for (uint32_t tile = g.tile0; tile < g.tile1; tile++, i++) {
          if (tile + 1 < g.tile1) scores(i + 1);
          wait(&sm.pfull[i & 1], i >> 1);
          wait(&sm.vclean[i % kSlots], i / kSlots);
          tc_after();
          const uint64_t vb = vd + (i % kSlots) * kPart;
          const uint32_t a = tmem + 128 * (i & 1), d = tmem + 256 + 128 * (i & 1);
          if (wait.ok) {  // this tile's P V, from zero: the sum over tiles is made in registers, where it is rounded
#pragma unroll
            for (uint32_t k = 0; k < kTcTile / 16; k++) {
              const uint32_t at = a + 32 * (k / 2) + 8 * (k % 2);
              tc_mma_ts(leader, d, at, vb + k * (2048 >> 4), idesc_f16(HD, true), k > 0);
              tc_mma_ts(leader, d, at + 16, vb + k * (2048 >> 4), idesc_f16(HD, true), true);
            }
            tc_commit(leader, &sm.ofull[i & 1]);
            tc_commit(leader, &sm.vempty[i % kSlots]);
          }
          __syncwarp();
        }
      }
      // the MMAs in flight end before TMEM is given back
      tc_commit(leader, &sm.drain);
      wait.ok = true;
      wait(&sm.drain, 0);
      __syncwarp();
    }
  } else {
    // ---- softmax: a thread a row, warpgroup wg a quarter of the positions and 32 dims ----
    asm volatile("setmaxnreg.inc.sync.aligned.u32 104;");
    const uint32_t wg = warp >> 2, r = t & 127;
    const uint32_t lanes = (warp & 3) * 32 << 16;
    uint32_t i = 0;
    for (uint32_t seg = 0; next_segment<1, kManySoft>(sm.ring, seg, wait, g); seg++) {
      const uint32_t rows = min(kManyRows, g.nodes * p.g - g.block * kManyRows);
      // the last segment's products are done: Q may be written
      put_queries<HD, kManyRows, MMA>(p, g, rows, warp, sm.q[0], BL, Smem::kTileBytes, sm.factor);
      __syncwarp();
      if (lane == 0) mbar_arrive(&sm.qfull);
      named_sync<1, kManySoft>();
      const float factor = sm.factor[r];
      const bool work = (warp & 3) * 32 < rows;  // a warp whose rows are all past the last one keeps step only
      const uint32_t rr = g.block * kManyRows + r, nd = rr / p.g;
      const bool live = r < rows;
      float o[32], m = -INFINITY, l = 0.0f, corr = 1.0f;
#pragma unroll
      for (int d = 0; d < 32; d++) o[d] = 0.0f;
      // add the P V of tile n (the n-th of the run) to this thread's 32 dims; `tile` its number in the unit
      auto fold = [&](uint32_t n, uint32_t tile, uint64_t sees0, uint64_t sees1) {
        if (wg >= HD / 32) return;  // no dims
        wait(&sm.ofull[n & 1], n >> 1);
        __syncwarp();
        tc_after();
        if (work) {
          uint32_t v[32];
          tc_ld32(tmem + lanes + 256 + 128 * (n & 1) + wg * 32, v);
          tc_ld_wait(v);
#pragma unroll
          for (int d = 0; d < 32; d++) o[d] = fmaf(o[d], corr, __uint_as_float(v[d]));
          if ((tile + 1) * kTcTile > g.len) {
            // non-finite V elements of nodes that this row sees
#pragma unroll 1
            for (int x = 0; x < 4; x++)
#pragma unroll 1
              for (uint32_t left = sm.odd[n & 7][x] & (uint32_t)((x < 2 ? sees0 : sees1) >> (32 * (x & 1))); left;
                   left &= left - 1) {
                const int64_t at_row = kv_row(p.c, g.s, tile * kTcTile + 32 * x + __ffs(left) - 1);
                if (at_row < 0) continue;  // the words are old ones: a wait has run out
                const __half2 *vr =
                    reinterpret_cast<const __half2 *>(p.c.v + (size_t)g.kvh * p.c.head_stride + at_row + wg * 32);
#pragma unroll
                for (int d = 0; d < 16; d++) {
                  const float2 f = __half22float2(vr[d]);
                  if (!isfinite(f.x)) o[2 * d] += f.x;
                  if (!isfinite(f.y)) o[2 * d + 1] += f.y;
                }
              }
          }
        }
        __syncwarp();
        tc_before();
      };
      uint64_t sees0 = 0, sees1 = 0;  // of the tile that is folded next
      for (uint32_t tile = g.tile0; tile < g.tile1; tile++, i++) {
        const uint32_t sa = tmem + lanes + 128 * (i & 1) + 32 * wg;
        wait(&sm.sfull[i & 1], i >> 1);
        __syncwarp();
        tc_after();
        float corr1 = 1.0f;
        uint64_t now0 = 0, now1 = 0;
        if (work) {
          uint32_t v[32];
          tc_ld32(sa, v);
          const bool drafted = (tile + 1) * kTcTile > g.len;
          const uint64_t ok0 = (uint64_t)sm.valid[i & 7][0] | (uint64_t)sm.valid[i & 7][1] << 32;
          const uint64_t ok1 = (uint64_t)sm.valid[i & 7][2] | (uint64_t)sm.valid[i & 7][3] << 32;
          const bool masked = drafted || (ok0 & ok1) != ~0ull;
          now0 = ok0, now1 = ok1;
          if (drafted) {
            now0 &= seen(p, tile * kTcTile - g.len, live, nd, g.first);
            now1 &= seen(p, tile * kTcTile + 64 - g.len, live, nd, g.first);
          }
          tc_ld_wait(v);
          if (masked) {
            const uint32_t bits = (uint32_t)((wg < 2 ? now0 : now1) >> (32 * (wg & 1)));
#pragma unroll
            for (int e = 0; e < 32; e++)
              if (!((bits >> e) & 1)) v[e] = 0xFF800000u;  // -inf
          }
          float t4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
          for (int e = 0; e < 32; e += 8)
#pragma unroll
            for (int u = 0; u < 4; u++)
              t4[u] = fmaxf(t4[u], fmaxf(__uint_as_float(v[e + 2 * u]), __uint_as_float(v[e + 2 * u + 1])));
          // the row's other positions are the other warpgroups'
          sm.top[i & 1][r][wg] = fmaxf(fmaxf(t4[0], t4[1]), fmaxf(t4[2], t4[3]));
          group_sync(4 + (warp & 3));
          const float4 tops = *reinterpret_cast<const float4 *>(sm.top[i & 1][r]);
          // the factor is a power of two: the products are exact, so that no exponent below is above that of the maximum
          const float mn = fmaxf(m, fmaxf(fmaxf(tops.x, tops.y), fmaxf(tops.z, tops.w)) * factor);
          corr1 = m == mn ? 1.0f : ex2(m - mn);
          m = mn;
          const float sub = mn == -INFINITY ? 0.0f : shifted(mn);
          float part[4] = {0.f, 0.f, 0.f, 0.f};
          uint32_t w[32];  // 16 words of parts, 16 of remainders
#pragma unroll
          for (int e = 0; e < 32; e += 2) {
            const float p0 = ex2(fmaf(__uint_as_float(v[e]), factor, -sub));
            const float p1 = ex2(fmaf(__uint_as_float(v[e + 1]), factor, -sub));
            part[(e / 2) & 3] += p0 + p1;
            split_f16(p0, p1, w[e / 2], w[16 + e / 2]);
          }
          tc_st32(sa, w);
          l = l * corr1 + ((part[0] + part[1]) + (part[2] + part[3]));
          asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
        }
        tc_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&sm.pfull[i & 1]);
        // the tile before, whose P V ran meanwhile
        if (tile > g.tile0) fold(i - 1, tile - 1, sees0, sees1);
        corr = corr1, sees0 = now0, sees1 = now1;
      }
      fold(i - 1, g.tile1 - 1, sees0, sees1);
      // the four quarters' sums of weights
      sm.ml[wg][r] = l;
      named_sync<1, kManySoft>();
      const float L = (sm.ml[0][r] + sm.ml[1][r]) + (sm.ml[2][r] + sm.ml[3][r]);
      const bool whole = g.whole();
      const size_t slot = g.slot;
      const float scale = whole ? (L != 0.0f ? 1.0f / L : 0.0f) : 1.0f;
      // whole units go to their rows of out; parts lie [hd / 4][row] float4
      float *dst = whole ? p.out + ((size_t)(g.first + (live ? nd : 0)) * p.h + g.kvh * p.g + rr % p.g) * HD + wg * 32
                         : p.part_o + ((slot * (HD / 4) + wg * 8) * kManyRows + r) * 4;
      const uint32_t step = whole ? 4 : 4 * kManyRows;
      if (live && wg < HD / 32) {
#pragma unroll
        for (int d = 0; d < 32; d += 4)
          *reinterpret_cast<float4 *>(dst + (size_t)(d / 4) * step) =
              make_float4(o[d] * scale, o[d + 1] * scale, o[d + 2] * scale, o[d + 3] * scale);
        if (!whole && wg == 0) {
          p.part_ml[(slot * kManyRows + r) * 2] = m;
          p.part_ml[(slot * kManyRows + r) * 2 + 1] = L;
        }
      }
      if (g.tile0 == 0 && t == 0) note_unit(p, g);
      named_sync<1, kManySoft>();  // Q and the sums may be written again
    }
  }
  tc_before();
  __syncthreads();
  if (warp == MMA) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512));
}

}  // namespace
