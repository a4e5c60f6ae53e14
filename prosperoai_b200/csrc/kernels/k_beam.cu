// Beam search's selection: the n_out best of beams x vocabulary candidates
// of every prompt, one launch, the logits read once.
//
//   score(b, t) = start_b + (x_t - m_b) - log Z_b,   Z_b = sum_t e^(x_t - m_b)
//
// Within a beam the order of the scores is the order of the logits, so a CTA
// needs neither m_b nor Z_b to know which of its logits can be chosen: it
// keeps the n_out largest of its slice, the slice's maximum and its sum of
// exponentials. The last CTA of a prompt to finish merges: m_b and Z_b of
// every beam from the slices in order, then the n_out best of the kept logits
// by score. What is added up is added in a fixed order; the chosen ones are
// ranked by (score, flat index), so nothing depends on which CTA is last.
//
// A slice is read in tiles of 4096 (16 registers a thread), the next one on
// its way while one is worked on. The n_out best of the first tile give a bar
// that few later logits reach; those that do go to a list of their warp, so
// that the warps meet at the first and the last tile only. The best of a tile
// or of the lists: every warp finds the ceil(n_out / 8)-th largest of its
// threads' maxima; the smallest of these is a bound that at least n_out
// values reach, and few others, which are collected and ranked.
//
// 16 prompts of 8 beams of 128256, 16 kept (66 MB, 10 us): 27 us, of which the
// reading and the exponentials 15, the first and last picks 5, the lists 4 and
// the merge 3. Before the merge kept its scores in registers between its two
// passes it was 30; of that form, 8192 logits a CTA, ranked there, took 40; a
// barrier a tile 39; four CTAs on an SM instead of three (64 registers, which
// spill) 33; tiles of 2048 41; three tiles ahead in shared memory 35; the
// lists by ballots 31.
//
// The exponentials are 2^((x - c) log2 e) with the thread's own c, at most 2
// below its maximum so far: x - c, the product and the constant are off by 2.5
// 2^-24 |x - c|, and the weighted mean of |x - c| is below that of |x - m| + 4,
// log(vocab) + 4 at most; 2^-22 each for the special function unit here and
// where c meets the slice's maximum; 6 additions in 32 bits, the others in 64.
// So log Z is off by less than 55 2^-24 at 128256 tokens.
#include <cuda_runtime.h>

#include <algorithm>
#include <cfloat>

#include "../b200_internal.h"
#include "b200_device.cuh"

namespace {

constexpr uint32_t kThreads = 256, kPer = 16, kTile = kThreads * kPer;  // logits of a CTA at a time: 16 registers a thread
constexpr uint32_t kCtasPerSm = 3, kSms = 148;
constexpr uint32_t kMaxPick = 64, kMaxBeams = 64, kMergeHold = 2, kCollect = 1024, kHold = 64;

struct BeamParams {
  const float *logits, *scores;
  const int32_t *done;
  uint64_t stride;
  uint32_t beams, vocab, slices, per, n_out;
  int32_t pad;
  float *out_scores;
  int32_t *out_parents, *out_tokens;
  float *top;      // scratch [row][slice]: the slice's maximum
  float *sum;      // scratch [row][slice]: its sum of e^(x - maximum)
  float *val;      // scratch [row][slice][n_out]: the kept logits, largest first, -inf behind them
  uint32_t *idx;   // scratch [row][slice][n_out]: their tokens
  uint32_t *cnt;   // counters [prompt], left at zero
};

template <typename T>
struct Cand {
  T v;
  uint32_t i;
};

// (value, index): larger first, equal values by the lower index
template <typename T>
__device__ __forceinline__ bool before(T v, uint32_t i, T w, uint32_t j) {
  return v > w || (v == w && i < j);
}

constexpr float kLog2e = 1.4426950408889634f;

// 2^x of the special function unit
__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

template <typename T>
__device__ __forceinline__ T ninf() {
  return -(T)INFINITY;
}

// The largest of the lanes' values.
__device__ __forceinline__ float warp_top(float v) {
  float top;
  asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(top) : "f"(v));
  return top;
}

// The `pick` first of the block's candidates into out[] (shared), ranked;
// `each` calls f(value, index) for every candidate of the calling thread that
// reaches a bound (others may be left out), the same each time; `most` is one
// of the thread's largest values, rounded to 32 bits (which keeps the order,
// so that a bound on rounded values holds).
// Candidates of value -inf are never taken. Returns how many there are (at
// most pick).
template <typename T, typename Each>
__device__ uint32_t block_pick(uint32_t pick, float most, Each each, Cand<T> *out, Cand<T> *buf) {
  __shared__ uint32_t count;
  __shared__ float bounds[kThreads / 32];
  __shared__ Cand<T> wbest[kThreads / 32];
  const uint32_t t = threadIdx.x, lane = t & 31;
  float left = most, nth = -INFINITY;
  for (uint32_t k = 0; k < (pick + kThreads / 32 - 1) / (kThreads / 32); k++) {
    nth = warp_top(left);
    if (lane == __ffs(__ballot_sync(0xffffffffu, left == nth)) - 1) left = -INFINITY;
  }
  __syncthreads();  // buf and out are free
  if (lane == 0) bounds[t >> 5] = nth;
  if (t == 0) count = 0;
  __syncthreads();
  float low = bounds[0];
#pragma unroll
  for (uint32_t w = 1; w < kThreads / 32; w++) low = fminf(low, bounds[w]);
  each([&](T v, uint32_t i) {
    if ((float)v >= low && v > ninf<T>()) {
      const uint32_t at = atomicAdd(&count, 1u);
      if (at < kCollect) buf[at] = Cand<T>{v, i};
    }
  }, low);
  __syncthreads();
  const uint32_t n = count;
  if (n <= kCollect) {
    for (uint32_t a = t; a < n; a += kThreads) {
      const Cand<T> me = buf[a];
      uint32_t r = 0;
#pragma unroll 4
      for (uint32_t b = 0; b < n; b++) r += before(buf[b].v, buf[b].i, me.v, me.i);
      if (r < pick) out[r] = me;
    }
    __syncthreads();
    return min(n, pick);
  }
  // many equal values: one after the other
  T lv = (T)INFINITY;
  uint32_t li = 0;
  for (uint32_t k = 0; k < pick; k++) {
    T bv = ninf<T>();
    uint32_t bi = 0xFFFFFFFFu;
    each([&](T v, uint32_t i) {
      if ((k == 0 || before(lv, li, v, i)) && v > ninf<T>() && before(v, i, bv, bi)) bv = v, bi = i;
    }, low);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const T ov = __shfl_xor_sync(0xffffffffu, bv, o);
      const uint32_t oi = __shfl_xor_sync(0xffffffffu, bi, o);
      if (before(ov, oi, bv, bi)) bv = ov, bi = oi;
    }
    if ((t & 31) == 0) wbest[t >> 5] = Cand<T>{bv, bi};
    __syncthreads();
    for (uint32_t w = 0; w < kThreads / 32; w++)
      if (before(wbest[w].v, wbest[w].i, bv, bi)) bv = wbest[w].v, bi = wbest[w].i;
    lv = bv, li = bi;
    if (t == 0) out[k] = Cand<T>{bv, bi};
    __syncthreads();
  }
  return pick;
}

// The next float above a value that is not NaN.
__device__ __forceinline__ float above(float v) { return nextafterf(v, INFINITY); }

// Keeps the M first of a warp's list of n > M entries (in order); returns the last one's value.
__device__ __noinline__ float warp_keep(Cand<float> *list, uint32_t n, uint32_t M) {
  const uint32_t lane = threadIdx.x & 31;
  float lv = INFINITY;
  for (uint32_t k = 0; k < M; k++) {  // the first of entries k .. n - 1 changes places with entry k
    float bv = -INFINITY;
    uint32_t bi = 0xFFFFFFFFu, at = 0;
    for (uint32_t a = k + lane; a < n; a += 32)
      if (before(list[a].v, list[a].i, bv, bi)) bv = list[a].v, bi = list[a].i, at = a;
    lv = warp_top(bv);
    const uint32_t i = __reduce_min_sync(0xffffffffu, bv == lv ? bi : 0xFFFFFFFFu);
    if (bv == lv && bi == i) {
      list[at] = list[k];
      list[k] = Cand<float>{lv, i};
    }
    __syncwarp();
  }
  return lv;
}

__global__ void __launch_bounds__(kThreads, kCtasPerSm) k_beam_select(BeamParams p) {
  pdl_trigger();
  pdl_wait();
  // what a pick collects (of 16 bytes in the merge), then the warps' lists
  __shared__ __align__(16) Cand<float> shared[kCollect + kThreads / 32 * (kHold + kPer * 32)];
  Cand<double> *buf_d = reinterpret_cast<Cand<double> *>(shared);
  __shared__ Cand<double> out_d[kMaxPick];
  __shared__ double logz[kMaxBeams], start[kMaxBeams];
  __shared__ float topb[kMaxBeams];
  __shared__ float redf[kThreads / 32];
  __shared__ double redd[kThreads / 32];
  __shared__ uint32_t ticket, counts[kThreads / 32];
  const uint32_t t = threadIdx.x, lane = t & 31, warp = t >> 5, slice = blockIdx.x, row = blockIdx.y, prompt = row / p.beams;
  const uint32_t M = p.n_out;
  const uint64_t slot = (uint64_t)row * p.slices + slice;
  const bool done = p.done && p.done[row] != 0;
  if (!done) {
    Cand<float> *buf = reinterpret_cast<Cand<float> *>(shared), *list = buf + kCollect + warp * (kHold + kPer * 32);
    Cand<float> *out = reinterpret_cast<Cand<float> *>(out_d);
    const uint32_t begin = slice * p.per, hi = min(p.vocab, begin + p.per);
    const float *x = p.logits + (uint64_t)row * p.stride;
    const bool wide = ((uintptr_t)x & 15) == 0;
    // thread t has logits lo + 4t .. +3 of a tile, then 1024 further on: v[e] is logit lo + (e/4) 1024 + 4t + e%4. In a
    // tile that is not full neighbours go to different warps: a warp with few logits would spoil the bound (9 x 13 beams
    // of 900 logits, 26 kept: 64 us, 13.4 now).
    float v[kPer], ahead[kPer];
    auto place = [&](uint32_t lo) { return hi - lo < kTile ? lane * (kThreads / 32) + warp : t; };
    auto load = [&](uint32_t lo) {
      const uint32_t tq = place(lo);
#pragma unroll
      for (uint32_t e = 0; e < kPer; e += 4) {
        const uint32_t i = lo + (e / 4) * (kThreads * 4) + 4 * tq;
        if (wide && i + 4 <= hi) {
          const float4 f = __ldcs(reinterpret_cast<const float4 *>(x + i));
          ahead[e] = f.x, ahead[e + 1] = f.y, ahead[e + 2] = f.z, ahead[e + 3] = f.w;
        } else {
#pragma unroll
          for (uint32_t q = 0; q < 4; q++) ahead[e + q] = i + q < hi ? x[i + q] : -INFINITY;
        }
      }
    };
    load(begin);
    float m = -INFINITY;         // the thread's maximum so far
    float c = -INFINITY;         // what its sum is relative to: m - 2 < c <= m
    double z = 0.0;              // sum of e^(x - c)
    float bar = -FLT_MAX;        // M logits of earlier tiles are above or equal but earlier: a later one has to reach it
    uint32_t n = 0, held = 0;    // the slice's best at the end; entries of the warp's list
    for (uint32_t lo = begin; lo < hi; lo += kTile) {
      float most = -INFINITY, quad[kPer / 4];
#pragma unroll
      for (uint32_t e = 0; e < kPer; e++) {
        v[e] = fmaxf(ahead[e], -INFINITY);  // drops NaN, which counts as -inf
        quad[e / 4] = e % 4 ? fmaxf(quad[e / 4], v[e]) : v[e];
      }
#pragma unroll
      for (uint32_t g = 0; g < kPer / 4; g++) most = fmaxf(most, quad[g]);
      const bool last = hi - lo <= kTile;
      if (!last) load(lo + kTile);
      m = fmaxf(m, most);
      if (most > c + 2.0f) {
        z *= exp2_fast((c - most) * kLog2e);
        c = most;
      }
      float part[4] = {0.0f, 0.0f, 0.0f, 0.0f};
      if (c == INFINITY) {
#pragma unroll
        for (uint32_t e = 0; e < kPer; e++) part[e & 3] += v[e] == INFINITY ? 1.0f : 0.0f;
      } else if (c > -INFINITY) {
#pragma unroll
        for (uint32_t e = 0; e < kPer; e++) part[e & 3] += exp2_fast((v[e] - c) * kLog2e);
      }
      z += (part[0] + part[1]) + (part[2] + part[3]);
      if (lo != begin && !last) {  // what passes the bar joins the warp's list
        if (!__any_sync(0xffffffffu, most >= bar)) continue;
        if (most >= bar) {
#pragma unroll
          for (uint32_t e = 0; e < kPer; e++)
            if (v[e] >= bar) list[atomicAdd(&counts[warp], 1u)] = Cand<float>{v[e], lo + (e / 4) * (kThreads * 4) + 4 * t + e % 4};
        }
        __syncwarp();
        held = *(volatile uint32_t *)&counts[warp];
        if (held > kHold) {
          bar = above(warp_keep(list, held, M)), held = M;
          if (lane == 0) counts[warp] = M;
        }
        __syncwarp();
        continue;
      }
      // the M best of the lists and of this tile
      const uint32_t tq = place(lo);
      for (uint32_t a = lane; a < held; a += 32) most = fmaxf(most, list[a].v);
      n = block_pick<float>(
          M, most,
          [&](auto f, float) {
#pragma unroll
            for (uint32_t e = 0; e < kPer; e++) f(v[e], lo + (e / 4) * (kThreads * 4) + 4 * tq + e % 4);
            for (uint32_t a = lane; a < held; a += 32) f(list[a].v, list[a].i);
          },
          out, buf);
      if (!last) {
        bar = n == M ? above(out[M - 1].v) : -FLT_MAX;
        held = n > warp ? (n - warp + kThreads / 32 - 1) / (kThreads / 32) : 0;
        if (lane == 0) counts[warp] = held;
        if (lane < held) list[lane] = out[lane * (kThreads / 32) + warp];
        __syncwarp();
      }
    }
    for (uint32_t k = t; k < M; k += kThreads) {
      p.val[slot * M + k] = k < n ? out[k].v : -INFINITY;
      p.idx[slot * M + k] = k < n ? out[k].i : 0;
    }
    const float mt = warp_top(m);
    if (lane == 0) redf[warp] = mt;
    __syncthreads();
    m = redf[0];
#pragma unroll
    for (uint32_t w = 1; w < kThreads / 32; w++) m = fmaxf(m, redf[w]);
    if (c != m) z *= exp2_fast((c - m) * kLog2e);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) z += __shfl_xor_sync(0xffffffffu, z, o);
    if (lane == 0) redd[warp] = z;
    if (t == 0) p.top[slot] = m;
  }
  // the last CTA of the prompt merges
  __syncthreads();
  if (t == 0) {
    if (!done) {
      double z = 0.0;
      for (uint32_t w = 0; w < kThreads / 32; w++) z += redd[w];
      p.sum[slot] = (float)z;
    }
    __threadfence();  // behind the barrier: for what the whole CTA wrote
    ticket = atomicAdd(&p.cnt[prompt], 1u);
  }
  __syncthreads();
  if (ticket != p.beams * p.slices - 1) return;
  __threadfence();
  const uint64_t row0 = (uint64_t)prompt * p.beams;
  for (uint32_t b = warp; b < p.beams; b += kThreads / 32) {  // a warp a beam, its slices in order
    const uint64_t r = (row0 + b) * p.slices;
    const bool over = p.done && p.done[row0 + b] != 0;
    const float first = p.scores[row0 + b];
    float m = -INFINITY;
    double z = 0.0;
    if (!over) {
      float mk = -INFINITY, sk = 0.0f;  // a lane's first slice, maximum and sum on their way at once
      if (lane < p.slices) mk = __ldcg(&p.top[r + lane]), sk = __ldcg(&p.sum[r + lane]);
      m = mk;
      for (uint32_t k = lane + 32; k < p.slices; k += 32) m = fmaxf(m, __ldcg(&p.top[r + k]));
      m = warp_max(m);
      for (uint32_t k = lane;;) {
        if (mk > -INFINITY) z += (double)sk * (mk == m ? 1.0 : exp((double)mk - (double)m));
        if ((k += 32) >= p.slices) break;
        mk = __ldcg(&p.top[r + k]), sk = __ldcg(&p.sum[r + k]);
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) z += __shfl_xor_sync(0xffffffffu, z, o);
    }
    if (lane == 0) {
      start[b] = first;
      topb[b] = m;
      logz[b] = over ? NAN : log(z);  // NaN marks a finished beam
    }
  }
  __syncthreads();
  // Candidates: beam b's kept logits, or the one of a finished beam, as (score, b * vocab + token). They lie in lists, one
  // a beam and slice, best first. The first 512, taken rank by rank, are a thread's to keep: neighbours go to different
  // warps, so that every warp has a part of each beam's best and its maxima are a bound that few others reach. Of the
  // other ranks a list is followed for as long as it reaches that bound (13 beams of 128256, 26 kept: 57 us with all of
  // them looked at, 18.5 now; 64 beams of 40000, 64 kept: 108 and 35).
  const uint32_t mine = (t & 31) * (kThreads / 32) + (((t >> 5) + t) & (kThreads / 32 - 1));
  const uint32_t lists = p.beams * p.slices, all = lists * M;
  auto score = [&](uint32_t list, uint32_t k, double &sc, uint32_t &flat) {
    const uint32_t b = list / p.slices;
    sc = ninf<double>();
    flat = 0;
    if (logz[b] != logz[b]) {
      if (k == 0 && list == b * p.slices) {
        sc = start[b];
        flat = b * p.vocab + (uint32_t)p.pad;
      }
    } else {
      const uint64_t at = (row0 * p.slices + list) * M + k;
      const float x = __ldcg(&p.val[at]);
      if (x > -INFINITY) {
        sc = start[b] + ((x == topb[b] ? 0.0 : (double)x - (double)topb[b]) - logz[b]);
        flat = b * p.vocab + __ldcg(&p.idx[at]);
      }
    }
    if (sc != sc) sc = ninf<double>();
  };
  double kept[kMergeHold];
  uint32_t flats[kMergeHold];
  float most = -INFINITY;
#pragma unroll
  for (uint32_t u = 0; u < kMergeHold; u++) {
    const uint32_t c = mine + u * kThreads;
    kept[u] = ninf<double>(), flats[u] = 0;
    if (c < all) score(c % lists, c / lists, kept[u], flats[u]);
    most = fmaxf(most, (float)kept[u]);
  }
  const uint32_t n = block_pick<double>(
      M, most,
      [&](auto f, float low) {
#pragma unroll
        for (uint32_t u = 0; u < kMergeHold; u++) f(kept[u], flats[u]);
        if (all <= kMergeHold * kThreads) return;
        for (uint32_t list = t; list < lists; list += kThreads) {
          uint32_t k = list < kMergeHold * kThreads ? (kMergeHold * kThreads - list + lists - 1) / lists : 0;
          for (; k < M; k++) {
            double sc;
            uint32_t flat;
            score(list, k, sc, flat);
            if ((float)sc < low) break;
            f(sc, flat);
          }
        }
      },
      out_d, buf_d);
  for (uint32_t k = t; k < M; k += kThreads) {
    const uint64_t o = (uint64_t)prompt * M + k;
    const bool is = k < n && out_d[k].v > ninf<double>();
    p.out_scores[o] = is ? (float)out_d[k].v : -INFINITY;
    p.out_parents[o] = is ? (int32_t)(row0 + out_d[k].i / p.vocab) : -1;
    p.out_tokens[o] = is ? (int32_t)(out_d[k].i % p.vocab) : p.pad;
  }
  if (t == 0) p.cnt[prompt] = 0;
}

}  // namespace

extern "C" pai_status_t pai_b200_beam_select_f32(pai_b200_ctx_t *ctx, uint64_t prompts, uint64_t beams, uint64_t vocab,
                                                 const float *logits, uint64_t stride, const float *scores,
                                                 const int32_t *done, int32_t pad, uint64_t n_out, float *out_scores,
                                                 int32_t *out_parents, int32_t *out_tokens) {
  if (!ctx || !logits || !scores || !out_scores || !out_parents || !out_tokens)
    return b200_fail(PAI_ERR_INVALID_ARG, "beam_select: NULL");
  if (prompts == 0 || beams == 0 || vocab == 0 || n_out == 0)
    return b200_fail(PAI_ERR_INVALID_ARG, "beam_select: a size is 0");
  if (stride < vocab)
    return b200_fail(PAI_ERR_MISMATCH, "beam_select: stride %llu below the vocabulary of %llu",
                     (unsigned long long)stride, (unsigned long long)vocab);
  if (pad < 0 || (uint64_t)pad >= vocab)
    return b200_fail(PAI_ERR_INVALID_ARG, "beam_select: pad token %d outside vocab %llu", pad, (unsigned long long)vocab);
  if (beams > kMaxBeams || n_out > kMaxPick)
    return b200_fail(PAI_ERR_UNSUPPORTED, "beam_select: %llu beams, %llu picked (at most %u and %u)",
                     (unsigned long long)beams, (unsigned long long)n_out, kMaxBeams, kMaxPick);
  // flat indexes within a prompt and the grid's rows stay in 32 and 16 bits
  if (vocab > 0x7FFFFFFFull / kMaxBeams || prompts > 65535 || prompts * beams > 65535)
    return b200_fail(PAI_ERR_UNSUPPORTED, "beam_select: %llu prompts of %llu beams over %llu tokens",
                     (unsigned long long)prompts, (unsigned long long)beams, (unsigned long long)vocab);
  if ((uintptr_t)logits & 3) return b200_fail(PAI_ERR_INVALID_ARG, "beam_select: logits must be 4-byte aligned");
  BeamParams p{};
  p.logits = logits, p.scores = scores, p.done = done, p.stride = stride, p.pad = pad;
  p.beams = (uint32_t)beams, p.vocab = (uint32_t)vocab, p.n_out = (uint32_t)n_out;
  const uint64_t rows = prompts * beams;
  // slices of whole tiles, as many as the CTAs that the GPU holds at a time leave for a row
  const uint64_t tiles = (vocab + kTile - 1) / kTile;
  const uint64_t share = std::clamp<uint64_t>((uint64_t)kCtasPerSm * kSms / rows, 1, tiles);
  p.per = (uint32_t)((tiles + share - 1) / share) * kTile;
  p.slices = (uint32_t)((vocab + p.per - 1) / p.per);
  p.out_scores = out_scores, p.out_parents = out_parents, p.out_tokens = out_tokens;
  const CtxDeviceGuard on(ctx);
  if (on.status()) return on.status();
  const uint64_t slots = rows * p.slices;
  float *scratch;
  pai_status_t st = b200_ctx_scratch(ctx, slots * (2 + 2 * n_out), (uint32_t)prompts, &scratch, &p.cnt);
  if (st) return st;
  p.top = scratch;
  p.sum = scratch + slots;
  p.val = scratch + 2 * slots;
  p.idx = (uint32_t *)(p.val + slots * n_out);
  b200_launch(ctx, k_beam_select, dim3(p.slices, (uint32_t)rows), dim3(kThreads), 0, p);
  return b200_launched(ctx, 1, "k_beam_select");
}
