// Tree attention on the fifth-generation tensor cores (tcgen05): what its two kernels share.
//
// Key tiles of 128 positions, whatever the rows: K and V come by tensor copies (TMA) in the 128-byte swizzle, a page or
// a share of one at a time; products go to TMEM. Both kernels are one CTA an SM and keep their roles in warps of their
// own, which meet at mbarriers; every wait is bounded.
#pragma once
#include <cuda.h>  // CUtensorMap and its enums (types only; the encoder comes from the runtime)

#include "attn_tree.cuh"

namespace {

constexpr uint32_t kTcTile = 128, kTcGrid = 148, kRing = 16;
// What a unit's start costs, in tiles: its queries, first maxima and output. The cut counts them, or a CTA that gets ten
// units of one tile each takes as long as 40 tiles of one unit (8 sequences of 5 to 5001 positions: 109 to 49 us).
constexpr uint32_t kStart = 3;

__device__ __forceinline__ uint64_t desc_k(uint32_t saddr) {  // K-major, 128-byte swizzle, 8-row groups of 1024 bytes
  return (uint64_t)((saddr >> 4) & 0x3FFFu) | (uint64_t)1u << 16 | (uint64_t)(1024u >> 4) << 32 | (uint64_t)1u << 46 |
         (uint64_t)2u << 61;
}
__device__ __forceinline__ uint64_t desc_mn(uint32_t saddr, uint32_t block) {
  // MN-major: 64-element blocks of the contiguous dimension `block` bytes apart, 8-row groups of 1024 bytes
  return (uint64_t)((saddr >> 4) & 0x3FFFu) | (uint64_t)(block >> 4) << 16 | (uint64_t)(1024u >> 4) << 32 |
         (uint64_t)1u << 46 | (uint64_t)2u << 61;
}
// kind::f16: fp16 A and B, fp32 sums, M = 128, N = n; a_mn, b_mn: that operand is MN-major
__host__ __device__ constexpr uint32_t idesc_f16(uint32_t n, bool b_mn, bool a_mn = false) {
  return (1u << 4) | (a_mn ? 1u << 15 : 0u) | (b_mn ? 1u << 16 : 0u) | ((n >> 3) << 17) | ((128u >> 4) << 24);
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
// Wait for the loads; the words pass through, so that nothing that uses them is moved before the wait.
__device__ __forceinline__ void tc_ld8(uint32_t at, uint32_t *r) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
               : "r"(at));
}
__device__ __forceinline__ void tc_ld_wait8(uint32_t *r) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7])
               :
               : "memory");
}
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
__device__ __forceinline__ void tc_st32(uint32_t at, const uint32_t *r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%32], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,"
      "%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31};" ::"r"(r[0]),
      "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]),
      "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]),
      "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]),
      "r"(r[29]), "r"(r[30]), "r"(r[31]), "r"(at)
      : "memory");
}
__device__ __forceinline__ void group_sync(uint32_t id) {  // of 128 threads
  __syncwarp();
  asm volatile("bar.sync %0, 128;" ::"r"(id) : "memory");
}
template <int ID, int N>
__device__ __forceinline__ void named_sync() {
  __syncwarp();
  asm volatile("bar.sync %0, %1;" ::"n"(ID), "n"(N) : "memory");
}

// A part of a unit: what the roles of a CTA work through, in order. `tile1` 0: there are no more.
struct Segment {
  uint32_t s, kvh, block, tile0, tile1, tiles;  // sequence, unit, key tiles of the part and of the unit
  uint32_t len, nodes, first;                   // the sequence's committed positions, nodes, first row
  uint32_t slot;                                // where a part is put
  uint32_t parts, slot0;                        // chunks that share the unit, slot of the first of its parts
  __device__ __forceinline__ bool whole() const { return tile0 == 0 && tile1 == tiles; }
};
// The warp that copies K walks over the pairs and hands the segments to the other roles through a ring: the divisions
// and lookups of a step are made once, and ahead. (A role is at most a few tiles behind it, never kRing segments.)
struct Ring {
  Segment seg[kRing];
  uint64_t full[kRing];
};

// upto[s]: (unit, tile) pairs of the sequences before s, each unit counted with kStart tiles more than it has (the caller
// bounds their sum). Every thread of the block calls
// it; a barrier must follow.
template <uint32_t MR, uint32_t THREADS>
__device__ __forceinline__ void pairs_before32(const TreeParams &p, uint32_t *upto) {
  const uint32_t n_seq = p.c.n_seq, lane = threadIdx.x & 31;
  for (uint32_t s = threadIdx.x; s < n_seq; s += THREADS) {
    const SeqWork w = seq_work<MR, kTcTile>(p, s);
    upto[s + 1] = w.blocks * (w.tiles + kStart) * p.c.hk;
  }
  if (threadIdx.x == 0) upto[0] = 0;
  if (n_seq <= 1) return;
  __syncthreads();
  if (threadIdx.x < 32) {
    uint32_t sum = 0;
    for (uint32_t s0 = 0; s0 < n_seq; s0 += 32) {
      const uint32_t s = s0 + lane;
      uint32_t x = s < n_seq ? upto[s + 1] : 0;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const uint32_t y = __shfl_up_sync(0xffffffffu, x, o);
        if (lane >= (uint32_t)o) x += y;
      }
      x += sum;
      if (s < n_seq) upto[s + 1] = x;
      sum = __shfl_sync(0xffffffffu, x, 31);
    }
  }
}

// Which of the 64 positions from node `base32` (negative: committed) on a row of node `nd` may see.
__device__ __forceinline__ uint64_t seen(const TreeParams &p, uint32_t base32, bool live, uint32_t nd, uint32_t first) {
  const int32_t base = (int32_t)base32;
  const uint64_t past = low_bits(-(int64_t)base);
  if (!live) return past;
  if (!p.mask) return low_bits((int64_t)nd + 1 - base);
  return past | (window(p.mask + (size_t)(first + nd) * p.words, p.words, base) & ~past);
}

// Whether node `nd` of the sequence whose rows begin at `first` may see node n.
__device__ __forceinline__ bool sees_node(const TreeParams &p, uint32_t first, uint32_t nd, uint32_t n) {
  if (!p.mask) return n <= nd;
  return n < 64 * p.words && (p.mask[(size_t)(first + nd) * p.words + n / 64] >> (n % 64)) & 1;
}

// A bounded wait that a role makes. After one has run out the role goes on without waiting or copying, so that the
// barriers among its own threads still meet; the error word tells the host.
struct Waiter {
  uint64_t limit_ns;
  uint32_t *err;
  bool ok = true;
  __device__ __forceinline__ void operator()(uint64_t *bar, uint32_t parity) {
    if (ok && !mbar_wait(bar, parity & 1u, limit_ns)) {
      ok = false;
      atomicExch(err, 1u);
    }
  }
};

// Whether all threads of a role say so: a warp, or THREADS that meet at barrier BAR.
template <int BAR, int THREADS>
__device__ __forceinline__ bool all_of(bool mine) {
  if (THREADS == 32) return __all_sync(0xffffffffu, mine);
  uint32_t all;
  __syncwarp();
  asm volatile(
      "{\n .reg .pred p, q;\n setp.ne.u32 q, %1, 0;\n bar.red.and.pred p, %2, %3, q;\n selp.u32 %0, 1, 0, p;\n}\n"
      : "=r"(all)
      : "r"((uint32_t)mine), "n"(BAR), "n"(THREADS)
      : "memory");
  return all;
}
// The n-th segment of the CTA; false behind the last. After a wait has run out anywhere in the role, all of it stops
// here.
template <int BAR = 0, int THREADS = 32>
__device__ __forceinline__ bool next_segment(Ring &ring, uint32_t n, Waiter &wait, Segment &g) {
  wait(&ring.full[n % kRing], n / kRing);
  g = ring.seg[n % kRing];
  return all_of<BAR, THREADS>(wait.ok) && g.tile1 != 0;
}

// The cut of the pairs into a chunk for each CTA, of `size` (the last may be shorter, and some CTAs may have none).
// SMs do not read memory equally fast (with even chunks the slowest of 148 takes 112 us where the fastest takes 66, 8
// sequences of one token at 16384 positions), but more and smaller chunks, taken from a counter as they come, cost more
// than they even out: a new chunk waits for its queries and its first maxima (two for each CTA 125 us, six 142, one 109).
// The leading role: yields the CTA's segments and hands them on.
struct Lead {
  uint32_t size = 1, at = 0, end = 0, s = 0, n = 0;
  __device__ __forceinline__ void begin(const TreeParams &p, const uint32_t *upto) {
    const uint32_t all = upto[p.c.n_seq];
    size = max((all + gridDim.x - 1) / gridDim.x, 1u);
    at = min(blockIdx.x * size, all);
    end = min(at + size, all);
    for (uint32_t hi = p.c.n_seq; s < hi;) {  // the sequence of the first pair
      const uint32_t mid = (s + hi) / 2;
      if (upto[mid + 1] <= at) s = mid + 1; else hi = mid;
    }
  }
  template <uint32_t MR>
  __device__ __forceinline__ bool next(const TreeParams &p, const uint32_t *upto, Ring &ring, Segment &g) {
    const uint32_t lane = threadIdx.x & 31, chunk = blockIdx.x;
    g.tile1 = 0;
    while (at < end && g.tile1 == 0) {
      while (upto[s + 1] <= at) s++;
      const SeqWork w = seq_work<MR, kTcTile>(p, s);
      const uint32_t span = w.tiles + kStart, unit = (at - upto[s]) / span, unit0 = upto[s] + unit * span;
      const uint32_t unit1 = unit0 + span, real0 = unit0 + kStart, to = min(end, unit1);
      g.s = s, g.kvh = unit / w.blocks, g.block = unit % w.blocks;
      g.tile0 = at > real0 ? at - real0 : 0, g.tile1 = to > real0 ? to - real0 : 0, g.tiles = w.tiles;
      g.len = w.len, g.nodes = w.nodes, g.first = w.first;
      g.slot = 2 * chunk + (chunk * size >= real0 ? 0 : 1);  // the chunk's first part of a unit, or its last
      const uint32_t c0 = real0 / size, c1 = (unit1 - 1) / size;
      g.parts = c1 - c0 + 1;
      g.slot0 = 2 * c0 + (c0 * size >= real0 ? 0 : 1);
      at = to;
    }
    if (lane == 0) {
      ring.seg[n % kRing] = g;
      mbar_arrive(&ring.full[n % kRing]);
    }
    n++;
    return g.tile1 != 0;
  }
};
// Copies, one warp for all K tiles or all V tiles: a lane a chunk of p.chunk positions, which lie in one page. The warp
// of K (LEADS) also hands out the segments, and notes in `valid` which positions of a tile hold a row. SLOTS tiles are
// in flight.
template <int HD, uint32_t MR, uint32_t SLOTS, bool LEADS, uint32_t WM>
__device__ __forceinline__ void copy_tiles(const TreeParams &p, const CUtensorMap *map, const uint32_t *upto, Ring &ring,
                                           uint8_t *slot0, uint64_t *full, uint64_t *empty,
                                           uint32_t (*valid)[4]) {
  constexpr uint32_t BL = kTcTile * 128, BYTES = HD / 64 * BL;
  const uint32_t lane = threadIdx.x & 31, chunks = kTcTile / p.chunk, chunk = p.chunk, P = p.c.page_tokens;
  Waiter wait{p.wait_ns, p.err};
  Lead lead;
  if (LEADS) lead.begin(p, upto);
  Segment g;
  uint32_t i = 0;  // tiles so far
  // After a wait has run out the leading warp hands out nothing more: the entries that it would write may still be read.
  for (uint32_t n = 0; LEADS ? __all_sync(0xffffffffu, wait.ok) && lead.next<MR>(p, upto, ring, g)
                             : next_segment(ring, n, wait, g);
       n++) {
    const uint32_t total = g.len + g.nodes;
    // where the lane's chunk of a tile lies: page (n_pages for a hole, which reads zeros), first row; -1: behind the
    // last position, not copied
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
      const uint32_t sl = i % SLOTS;
      const int32_t at = page, r = row;
      find(tile + 1);  // the next tile's table entries come while this one is copied
      const uint32_t copied = __ballot_sync(0xffffffffu, at >= 0);
      const uint32_t there = __ballot_sync(0xffffffffu, at >= 0 && at < (int32_t)p.c.n_pages);
      if (i >= SLOTS) wait(&empty[sl], i / SLOTS - 1);
      __syncwarp();
      if (LEADS) {
        if (lane < 4) {  // the word of positions 32 lane .. + 31
          const uint32_t cap = min(total, p.c.max_pages * P), pos = tile * kTcTile + 32 * lane;
          uint32_t bits = 0;
          if (chunk >= 32) {
            bits = (there >> (32 * lane / chunk)) & 1 ? 0xFFFFFFFFu : 0u;
          } else {
            for (uint32_t c = 0; c < 32 / chunk; c++)
              if ((there >> (32 / chunk * lane + c)) & 1) bits |= ((1u << chunk) - 1) << (c * chunk);
          }
          valid[i & WM][lane] = bits & (uint32_t)low_bits((int64_t)cap - pos);
        }
        __syncwarp();
      }
      if (wait.ok) {
        uint8_t *dst = slot0 + sl * BYTES + lane * chunk * 128;
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
  wait.ok = true;
  for (uint32_t n = i < SLOTS ? 0 : i - SLOTS; n < i; n++) wait(&full[n % SLOTS], n / SLOTS);
}

// V tiles are handed on to the MMAs by WARPS warps (this one is `w`), after they have looked at the rows of those that
// hold nodes: a non-finite V row may only reach the rows that see its node, and a weight of 0 does not keep it out of a
// product. Such elements (those of stale rows behind the last node too) become 0 here, and `odd` tells where; they are
// added later to the rows that see them. (Every tile is handed on: a barrier that was watched for some phases only could
// be two phases on.)
template <int HD, uint32_t SLOTS, uint32_t WARPS, uint32_t WM>
__device__ __forceinline__ void clean_tiles(const TreeParams &p, Ring &ring, uint32_t w, uint8_t *slot0, uint64_t *full,
                                            uint64_t *clean, uint32_t (*odd)[4]) {
  constexpr uint32_t BL = kTcTile * 128, BYTES = HD / 64 * BL, CH = HD / 8;
  const uint32_t lane = threadIdx.x & 31;
  Waiter wait{p.wait_ns, p.err};
  Segment g;
  uint32_t i = 0;
  for (uint32_t n = 0; next_segment(ring, n, wait, g); n++)
    for (uint32_t tile = g.tile0; tile < g.tile1; tile++, i++) {
      const uint32_t sl = i % SLOTS;
      wait(&full[sl], i / SLOTS);
      __syncwarp();
      if ((tile + 1) * kTcTile > g.len) {
        const uint32_t skip = g.len > tile * kTcTile ? g.len - tile * kTcTile : 0;  // committed rows of the tile
#pragma unroll 1
        for (uint32_t x = w; x < 4; x += WARPS) {  // a lane has a row of each 32
          const uint32_t r = 32 * x + lane;
          bool bad = false;
          if (r >= skip) {
            uint8_t *row = slot0 + sl * BYTES + r * 128;
#pragma unroll 8
            for (uint32_t ch = 0; ch < CH; ch++) {
              uint4 *at = reinterpret_cast<uint4 *>(row + (ch / 8) * BL + (((ch % 8) ^ (r & 7)) << 4));
              uint4 v = *at;
              // an exponent of all ones carries into the sign's place
              const uint32_t E = 0x7C007C00u, one = 0x04000400u;
              if ((((v.x & E) + one) | ((v.y & E) + one) | ((v.z & E) + one) | ((v.w & E) + one)) & 0x80008000u) {
                bad = true;
                uint32_t *cw = reinterpret_cast<uint32_t *>(&v);
#pragma unroll
                for (int y = 0; y < 4; y++) {
                  if ((cw[y] & 0x7C00u) == 0x7C00u) cw[y] &= 0xFFFF0000u;
                  if ((cw[y] & 0x7C000000u) == 0x7C000000u) cw[y] &= 0xFFFFu;
                }
                *at = v;
              }
            }
          }
          const uint32_t word = __ballot_sync(0xffffffffu, bad);
          if (lane == 0) odd[i & WM][x] = word;
        }
        fence_proxy_async();
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&clean[sl]);
    }
}

// Query rows, with the scores' scale, into shared memory as a K-major operand [64 dims][rows][128 bytes], a power of two
// and two fp16 parts a row: warp `w` of WARPS has MR / WARPS rows; the remainders lie `rem` bytes behind the parts.
template <int HD, uint32_t MR, uint32_t WARPS>
__device__ __forceinline__ void put_queries(const TreeParams &p, const Segment &g, uint32_t rows, uint32_t w, uint8_t *q,
                                            uint32_t block, uint32_t rem, float *factor) {
  constexpr uint32_t LR = HD / 4, RW = 32 / LR, WR = MR / WARPS;  // lanes of a row, rows of an access, rows of a warp
  constexpr uint32_t UN = WR / RW < 4 ? WR / RW : 4;
  const uint32_t lane = threadIdx.x & 31, d4 = lane % LR;
#pragma unroll 1
  for (uint32_t b0 = 0; b0 < WR; b0 += UN * RW) {
    float4 f[UN];
#pragma unroll
    for (uint32_t u = 0; u < UN; u++) {
      const uint32_t rl = w * WR + b0 + u * RW + lane / LR, rr = g.block * MR + rl;
      f[u] = rl < rows ? *reinterpret_cast<const float4 *>(
                             p.q + ((size_t)(g.first + rr / p.g) * p.h + g.kvh * p.g + rr % p.g) * HD + 4 * d4)
                       : make_float4(0.f, 0.f, 0.f, 0.f);
    }
#pragma unroll
    for (uint32_t u = 0; u < UN; u++) {
      const uint32_t rl = w * WR + b0 + u * RW + lane / LR;
      f[u].x *= p.scale, f[u].y *= p.scale, f[u].z *= p.scale, f[u].w *= p.scale;
      float top = fmaxf(fmaxf(fabsf(f[u].x), fabsf(f[u].y)), fmaxf(fabsf(f[u].z), fabsf(f[u].w)));
#pragma unroll
      for (uint32_t o = LR / 2; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
      float down, up;
      row_scale(top, down, up);
      uint2 hi, lo;
      split_f16(f[u].x * down, f[u].y * down, hi.x, lo.x);
      split_f16(f[u].z * down, f[u].w * down, hi.y, lo.y);
      const uint32_t at = (d4 / 16) * block + rl * 128 + (((d4 % 16) / 2 ^ (rl & 7)) << 4) + (d4 & 1) * 8;
      *reinterpret_cast<uint2 *>(q + at) = hi;
      *reinterpret_cast<uint2 *>(q + rem + at) = lo;
      if (d4 == 0) factor[rl] = up;
    }
  }
  fence_proxy_async();
}

// For the joining kernel: how many chunks hold parts of the unit (0: it is whole), and the first one's slot.
__device__ __forceinline__ void note_unit(const TreeParams &p, const Segment &g) {
  uint32_t *u = p.units + 2 * (((size_t)g.s * p.c.hk + g.kvh) * p.max_blocks + g.block);
  u[0] = g.whole() ? 0 : g.parts;
  u[1] = g.slot0;
}

// Join the parts of the units that several chunks shared: CTA (unit, 8 rows), a thread 4 dims of a row. Parts lie
// [row][hd] (BY_ROW) or [hd / 4][row] float4, as the kernels have them. What it takes (4.7 us by itself for a row of each
// of 64 units, 14 for 64 nodes of 8 sequences with 18 MB of parts) is the latency of loads that need one another: so the
// first 8 parts of a row are under way while the maxima and sums are read (90.1 to 89.0 us for one token at 131072;
// 4 or 16 parts, or 4 rows a CTA, are slower for one of few and many parts).
constexpr uint32_t kJoinRows = 8, kJoinParts = 8;
template <int HD, uint32_t MR, bool BY_ROW>
__global__ void __launch_bounds__(kJoinRows * HD / 4) k_attn_tree_join(TreeParams p) {
  pdl_trigger();
  pdl_wait();
  __shared__ float ws[kJoinRows][kTcGrid];
  __shared__ float inv[kJoinRows];
  const uint32_t unit = blockIdx.x, block = unit % p.max_blocks, kvh = unit / p.max_blocks % p.c.hk;
  const uint32_t s = unit / p.max_blocks / p.c.hk, row0 = blockIdx.y * kJoinRows, t = threadIdx.x;
  const uint2 made = reinterpret_cast<const uint2 *>(p.units)[unit];  // on its way together with the sequence's
  const SeqWork w = seq_work<MR, kTcTile>(p, s);
  if (block >= w.blocks) return;
  const uint32_t rows = min(MR, w.nodes * p.g - block * MR);
  const uint32_t parts = unit_parts(made.x, made.y, p.slots), first = made.y;
  if (parts == 0 || row0 >= rows) return;
  auto slot = [&](uint32_t q) -> size_t { return part_slot(first, q); };
  const uint32_t n = min(kJoinRows, rows - row0), warps = kJoinRows * HD / 128, lane = t & 31;
  const uint32_t r = BY_ROW ? t / (HD / 4) : t % kJoinRows, d4 = BY_ROW ? t % (HD / 4) : t / kJoinRows;
  float4 f[kJoinParts];
  auto load = [&](uint32_t q0) {
#pragma unroll
    for (uint32_t u = 0; u < kJoinParts; u++)
      if (q0 + u < parts)
        f[u] = *reinterpret_cast<const float4 *>(p.part_o + (BY_ROW ? (slot(q0 + u) * MR + row0 + r) * HD + 4 * d4
                                                                    : ((slot(q0 + u) * (HD / 4) + d4) * MR + row0 + r) * 4));
  };
  if (r < n) load(0);  // together with the maxima and sums
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
  if (r >= n) return;
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  for (uint32_t q0 = 0;;) {
#pragma unroll
    for (uint32_t u = 0; u < kJoinParts; u++)
      if (q0 + u < parts) {
        const float y = ws[r][q0 + u];
        acc.x = fmaf(f[u].x, y, acc.x), acc.y = fmaf(f[u].y, y, acc.y);
        acc.z = fmaf(f[u].z, y, acc.z), acc.w = fmaf(f[u].w, y, acc.w);
      }
    q0 += kJoinParts;
    if (q0 >= parts) break;
    load(q0);
  }
  const uint32_t rr = block * MR + row0 + r;
  const float y = inv[r];
  *reinterpret_cast<float4 *>(p.out + ((size_t)(w.first + rr / p.g) * p.h + kvh * p.g + rr % p.g) * HD + 4 * d4) =
      make_float4(acc.x * y, acc.y * y, acc.z * y, acc.w * y);
}

}  // namespace
