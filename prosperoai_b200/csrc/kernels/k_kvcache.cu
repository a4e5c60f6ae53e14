// Operators on a cache view: rotary append of drafted nodes, moving the
// accepted ones together, and forking sequences (page tables, partly filled
// pages, new pages; rows of a cache without pages).
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>

#include "../b200_internal.h"
#include "b200_device.cuh"
#include "kv_view.cuh"

namespace {

// ---- rotary append ---------------------------------------------------------------------------
// CTA (node, sequence, group of heads): hd/8 threads a head, 4 pairs (i, i +
// hd/2) each, so that every access is 16 bytes (8 of fp16). The products and
// sums are rounded one by one (rope_pair), as in the decode step. Bound by the
// launch and three loads that need one another: 4.7 us for 8 rows of 32 + 16
// heads of 128, 8.3 for 512 rows (21 MB, 3.2 us).
constexpr uint32_t kAppendThreads = 128;

struct AppendParams {
  KvDev c;
  uint32_t h, max_nodes;
  uint64_t rows, table_len;
  const int32_t *lens, *off, *depth;
  const float *qkv, *cos_t, *sin_t;
  float *q;
};

__device__ __forceinline__ void store_half4(__half *dst, const float (&v)[4]) {
  const __half2 a = __floats2half2_rn(v[0], v[1]), b = __floats2half2_rn(v[2], v[3]);
  uint2 w;
  w.x = *reinterpret_cast<const uint32_t *>(&a);
  w.y = *reinterpret_cast<const uint32_t *>(&b);
  *reinterpret_cast<uint2 *>(dst) = w;
}

__global__ void __launch_bounds__(kAppendThreads) k_rope_append(AppendParams p) {
  pdl_trigger();
  pdl_wait();
  const uint32_t hd = p.c.hd, r2 = hd / 2, tph = hd / 8;  // threads of a head
  const uint32_t s = blockIdx.y, i = blockIdx.x;
  const uint32_t head = blockIdx.z * (kAppendThreads / tph) + threadIdx.x / tph, j = (threadIdx.x % tph) * 4;
  if (threadIdx.x / tph >= kAppendThreads / tph || head >= p.h + 2 * p.c.hk) return;
  uint32_t first;
  const uint32_t n = kv_nodes(p.off, s, p.rows, p.max_nodes, &first);
  if (i >= n) return;
  const uint64_t row = (uint64_t)first + i;
  const uint32_t len = kv_len(p.c, p.lens, s);
  const int64_t at = (int64_t)len + (p.depth ? p.depth[row] : (int32_t)i);
  const bool turns = at >= 0 && (uint64_t)at < p.table_len;
  const float *x = p.qkv + (row * (p.h + 2 * p.c.hk) + head) * hd;
  float a[4], b[4];
  *reinterpret_cast<float4 *>(a) = *reinterpret_cast<const float4 *>(x + j);
  *reinterpret_cast<float4 *>(b) = *reinterpret_cast<const float4 *>(x + r2 + j);
  if (head < p.h + p.c.hk && turns) {
    float c[4], d[4];
    *reinterpret_cast<float4 *>(c) = *reinterpret_cast<const float4 *>(p.cos_t + at * r2 + j);
    *reinterpret_cast<float4 *>(d) = *reinterpret_cast<const float4 *>(p.sin_t + at * r2 + j);
#pragma unroll
    for (int e = 0; e < 4; e++) rope_pair(a[e], b[e], c[e], d[e], a[e], b[e]);
  }
  if (head < p.h) {
    if (!turns) {
#pragma unroll
      for (int e = 0; e < 4; e++) a[e] = b[e] = __int_as_float(0x7fffffff);
    }
    float *o = p.q + (row * p.h + head) * hd;
    *reinterpret_cast<float4 *>(o + j) = *reinterpret_cast<float4 *>(a);
    *reinterpret_cast<float4 *>(o + r2 + j) = *reinterpret_cast<float4 *>(b);
    return;
  }
  if (!turns) return;
  const int64_t at_row = kv_row(p.c, s, len + i);
  if (at_row < 0) return;
  const bool is_v = head >= p.h + p.c.hk;
  __half *dst = (is_v ? p.c.v : p.c.k) + at_row + (uint64_t)(head - p.h - (is_v ? p.c.hk : 0)) * p.c.head_stride;
  store_half4(dst + j, a);
  store_half4(dst + r2 + j, b);
}

// ---- accepted rows ---------------------------------------------------------------------------
// CTA (layer x plane, sequence): its columns are (kv head, 16 bytes of a
// row), one thread each. A path ascends, so a row's target never lies behind
// the sources of later rows: a thread reads kAcceptBatch rows of its column
// and then writes them, in path order, and needs no other thread. 6 rows of 8
// sequences in 32 layers of 8 heads of 128 (10 MB, 1.6 us): 6.2 us; a launch
// that moves nothing 5.0.
constexpr uint32_t kAcceptThreads = 128;
constexpr int kAcceptBatch = 8;

__global__ void __launch_bounds__(kAcceptThreads) k_kv_accept(KvDev c, uint32_t max_path, const int32_t *lens,
                                                              const int32_t *path, const int32_t *n_path,
                                                              int32_t *lens_out, uint32_t *cnt) {
  pdl_trigger();
  pdl_wait();
  extern __shared__ int64_t offs[];  // [max_path] sources, [max_path] targets
  __shared__ uint32_t keep;
  const uint32_t s = blockIdx.z, layer = blockIdx.x / 2;
  const uint32_t len = kv_len(c, lens, s);
  const int32_t np = n_path[s];
  const uint32_t n = np < 0 ? 0u : min((uint32_t)np, max_path);
  if (threadIdx.x == 0) keep = n;
  __syncthreads();
  const int32_t *pt = path + (size_t)s * max_path;
  for (uint32_t i = threadIdx.x; i < n; i += kAcceptThreads) {
    const int64_t e = pt[i], before = i ? pt[i - 1] : -1;
    const int64_t pos = (int64_t)len + e;
    const bool up = e > before && e >= (int64_t)i && pos <= 0x7FFFFFFF;
    const int64_t src = up ? kv_row(c, s, (uint32_t)pos) : -1, dst = up ? kv_row(c, s, len + i) : -1;
    offs[i] = src;
    offs[max_path + i] = dst;
    if (src < 0 || dst < 0) atomicMin(&keep, i);
  }
  __syncthreads();
  const uint32_t m = keep;
  const uint32_t chunks = c.hd / 8, cols = c.hk * chunks;
  __half *base = (blockIdx.x & 1 ? c.v : c.k) + (size_t)layer * c.layer_stride;
  for (uint32_t col = blockIdx.y * kAcceptThreads + threadIdx.x; col < cols; col += gridDim.y * kAcceptThreads) {
    __half *b = base + (col / chunks) * c.head_stride + (col % chunks) * 8;
    for (uint32_t i0 = 0; i0 < m; i0 += kAcceptBatch) {
      uint4 v[kAcceptBatch];
#pragma unroll
      for (int u = 0; u < kAcceptBatch; u++)
        if (i0 + u < m) v[u] = *reinterpret_cast<const uint4 *>(b + offs[i0 + u]);
#pragma unroll
      for (int u = 0; u < kAcceptBatch; u++)
        if (i0 + u < m && offs[i0 + u] != offs[max_path + i0 + u])
          *reinterpret_cast<uint4 *>(b + offs[max_path + i0 + u]) = v[u];
    }
  }
  // lens_out may be lens: it is written once every CTA of the sequence has read lens
  __syncthreads();
  if (threadIdx.x == 0) {
    const uint32_t all = gridDim.x * gridDim.y;
    __threadfence();
    if (atomicAdd(&cnt[s], 1u) == all - 1) {
      lens_out[s] = (int32_t)(len + m);
      cnt[s] = 0;
    }
  }
}

// ---- forks -----------------------------------------------------------------------------------
// One CTA plans: it reads the tables and lengths, writes the new table and
// lists the copies; a second kernel makes the copies. What a page is used
// for is a maximum (its rows in use) and a minimum (the first sequence that
// extends it), so the order of the atomics changes nothing. The copying kernel
// is launched beside the plan and waits for it. 8 beams, 4 of them copying a
// partly filled page in 32 layers (63 MB, 9.6 us): 18.5 us, 23.3 with one
// kernel behind the other; 8 runs of 700 positions (734 MB, 112 us): 119 us.
struct ForkCopy {
  int32_t src, dst;    // pages; without a table: the parent sequence, this sequence
  uint32_t from, rows; // rows [from, rows) of the page
};

struct ForkParams {
  KvDev c;
  uint32_t first, paged;
  const int32_t *lens, *parents, *grow;
  int32_t *table_out, *lens_out, *granted;
  int32_t *used, *keeper;  // scratch [n_pages]
  int32_t *fresh;          // scratch [want of all sequences]: the free pages, lowest first
  ForkCopy *copies;        // scratch [n_seq]
};

constexpr uint32_t kPlanThreads = 1024, kMaxSeq = 1024;

__device__ __forceinline__ uint32_t block_scan(uint32_t v, uint32_t *tmp, uint32_t *total) {
  // exclusive sums over the block's threads
  const uint32_t lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  uint32_t x = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint32_t y = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= (uint32_t)o) x += y;
  }
  __syncthreads();
  if (lane == 31) tmp[w] = x;
  __syncthreads();
  if (w == 0) {
    uint32_t t = tmp[lane];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint32_t y = __shfl_up_sync(0xffffffffu, t, o);
      if (lane >= (uint32_t)o) t += y;
    }
    tmp[lane] = t;
  }
  __syncthreads();
  *total = tmp[31];
  return x - v + (w ? tmp[w - 1] : 0);
}

__global__ void __launch_bounds__(kPlanThreads) k_kv_fork_plan(ForkParams p) {
  pdl_trigger();
  pdl_wait();
  const KvDev &c = p.c;
  __shared__ int32_t par[kMaxSeq];
  __shared__ uint32_t len[kMaxSeq];
  __shared__ uint32_t tmp[32];
  const uint32_t t = threadIdx.x, P = c.page_tokens, W = c.max_pages, n = c.n_seq;
  const uint64_t cap = (uint64_t)W * P;
  uint32_t g = 0, l = 0;
  if (t < n) {
    const int64_t q = p.parents ? p.parents[t] : (int32_t)t;
    const bool live = q >= 0 && q < (int64_t)n;
    l = live ? kv_len(c, p.lens, (uint32_t)q) : 0;
    const int32_t want = live && p.grow ? p.grow[t] : 0;
    g = want > 0 ? (uint32_t)want : 0;
    par[t] = live ? (int32_t)q : -1;
    len[t] = l;
  }
  const bool fits = (uint64_t)l + g <= cap;
  if (!p.paged) {
    __syncthreads();
    if (t < n) {
      p.lens_out[t] = (int32_t)l;
      p.granted[t] = fits ? (int32_t)g : 0;
      p.copies[t] = ForkCopy{par[t], (int32_t)t, p.first, par[t] == (int32_t)t ? 0u : l};
    }
    return;
  }
  for (uint32_t i = t; i < c.n_pages; i += kPlanThreads) {
    p.used[i] = 0;
    p.keeper[i] = 0x7FFFFFFF;
  }
  __syncthreads();
  for (uint64_t e = t; e < (uint64_t)n * W; e += kPlanThreads) {
    const uint32_t i = (uint32_t)(e / W), j = (uint32_t)(e % W);
    int32_t page = -1;
    if ((uint64_t)j * P < len[i]) {
      page = c.table[(size_t)par[i] * W + j];
      if ((uint32_t)page >= c.n_pages) page = -1;
      if (page >= 0) atomicMax(&p.used[page], (int32_t)min(P, len[i] - j * P));
    }
    p.table_out[e] = page;
  }
  __syncthreads();
  const uint32_t have = (l + P - 1) / P, mine = l % P;
  int32_t last = -1;
  if (t < n && mine) {
    last = c.table[(size_t)par[t] * W + have - 1];
    if ((uint32_t)last >= c.n_pages) last = -1;
  }
  const bool hole = mine && last < 0;
  if (t < n && g && last >= 0 && (int32_t)mine == p.used[last]) atomicMin(&p.keeper[last], (int32_t)t);
  __syncthreads();
  const bool able = t < n && g && fits && !hole;
  const bool copy = able && last >= 0 && p.keeper[last] != (int32_t)t;
  const uint32_t upto = able ? (uint32_t)(((uint64_t)l + g + P - 1) / P) : have;
  const uint32_t want = able ? upto - have + copy : 0;
  uint32_t all;
  const uint32_t begin = block_scan(want, tmp, &all);
  // the lowest free pages, as many as are wanted
  uint32_t found = 0;
  for (uint32_t i0 = 0; i0 < c.n_pages && found < all; i0 += kPlanThreads) {
    const uint32_t i = i0 + t;
    const uint32_t is_free = i < c.n_pages && p.used[i] == 0;
    uint32_t got;
    const uint32_t at = found + block_scan(is_free, tmp, &got);
    if (is_free && at < all) p.fresh[at] = (int32_t)i;
    found += got;
  }
  __syncthreads();
  if (t >= n) return;
  const bool ok = able && (!want || (uint64_t)begin + want <= found);
  p.lens_out[t] = (int32_t)l;
  p.granted[t] = ok ? (int32_t)g : 0;
  ForkCopy k{0, 0, 0, 0};
  if (ok) {
    uint32_t at = begin;
    if (copy) {
      k = ForkCopy{last, p.fresh[at], 0, mine};
      p.table_out[(size_t)t * W + have - 1] = p.fresh[at++];
    }
    for (uint32_t j = have; j < upto; j++) p.table_out[(size_t)t * W + j] = p.fresh[at++];
  }
  p.copies[t] = k;
}

// Copies of the plan's pages: CTA (layer x plane, sequence, share of the
// (kv head, row, 16 bytes) of a page).
constexpr uint32_t kCopyThreads = 256;
constexpr int kCopyBatch = 4;

__global__ void __launch_bounds__(kCopyThreads) k_kv_fork_pages(KvDev c, const ForkCopy *copies) {
  pdl_trigger();
  pdl_wait();
  const ForkCopy k = copies[blockIdx.y];
  if (k.rows == 0) return;
  const uint32_t layer = blockIdx.x / 2;
  __half *base = (blockIdx.x & 1 ? c.v : c.k) + (size_t)layer * c.layer_stride;
  const __half *src = base + (uint64_t)k.src * c.page_stride;
  __half *dst = base + (uint64_t)k.dst * c.page_stride;
  const uint32_t per = k.rows * (c.hd / 8);  // 16-byte pieces of a head's rows: they follow one another
  const uint64_t all = (uint64_t)per * c.hk, step = (uint64_t)gridDim.z * kCopyThreads;
  for (uint64_t i0 = (uint64_t)blockIdx.z * kCopyThreads + threadIdx.x; i0 < all; i0 += step * kCopyBatch) {
    uint4 v[kCopyBatch];
    uint64_t o[kCopyBatch];
#pragma unroll
    for (int u = 0; u < kCopyBatch; u++) {
      const uint64_t i = i0 + u * step;
      o[u] = (i / per) * c.head_stride + (i % per) * 8;
      if (i < all) v[u] = *reinterpret_cast<const uint4 *>(src + o[u]);
    }
#pragma unroll
    for (int u = 0; u < kCopyBatch; u++)
      if (i0 + u * step < all) *reinterpret_cast<uint4 *>(dst + o[u]) = v[u];
  }
}

// Rows of a cache without pages: a thread has one 16-byte column of every
// sequence, reads what the new sequences take from their parents, and then
// writes it, so that exchanges need no second buffer.
template <int NS>
__global__ void __launch_bounds__(kCopyThreads) k_kv_fork_runs(KvDev c, const ForkCopy *copies) {
  pdl_trigger();
  pdl_wait();
  __shared__ ForkCopy cp[NS];
  for (uint32_t i = threadIdx.x; i < NS; i += kCopyThreads) cp[i] = i < c.n_seq ? copies[i] : ForkCopy{0, 0, 0, 0};
  __syncthreads();
  uint32_t top = 0, from = 0;
#pragma unroll
  for (int i = 0; i < NS; i++) {
    top = max(top, cp[i].rows);
    from = max(from, cp[i].from);
  }
  if (top <= from) return;
  const uint32_t layer = blockIdx.x / 2, chunks = c.hd / 8, head = blockIdx.y;
  __half *base = (blockIdx.x & 1 ? c.v : c.k) + (size_t)layer * c.layer_stride + head * c.head_stride;
  const uint64_t end = (uint64_t)top * chunks;
  for (uint64_t e = (uint64_t)from * chunks + blockIdx.z * kCopyThreads + threadIdx.x; e < end;
       e += (uint64_t)gridDim.z * kCopyThreads) {
    const uint32_t row = (uint32_t)(e / chunks);
    uint4 v[NS];
#pragma unroll
    for (int i = 0; i < NS; i++)
      if (row < cp[i].rows) v[i] = *reinterpret_cast<const uint4 *>(base + (uint64_t)cp[i].src * c.page_stride + e * 8);
#pragma unroll
    for (int i = 0; i < NS; i++)
      if (row < cp[i].rows) *reinterpret_cast<uint4 *>(base + (uint64_t)cp[i].dst * c.page_stride + e * 8) = v[i];
  }
}

}  // namespace

extern "C" pai_status_t pai_b200_rope_append_f16kv(pai_b200_ctx_t *ctx, const pai_b200_kv_view_t *kv, uint32_t layer,
                                                   uint64_t h, uint64_t rows, uint32_t max_nodes, const int32_t *lens,
                                                   const int32_t *node_off, const int32_t *depth, const float *qkv,
                                                   const float *cos_t, const float *sin_t, uint64_t table_len,
                                                   float *q_out) {
  AppendParams p{};
  if (!ctx) return b200_fail(PAI_ERR_INVALID_ARG, "rope_append: NULL context");
  pai_status_t st = kv_nodes_check(kv, "rope_append", layer, h, rows, max_nodes, lens, node_off, p.c);
  if (st) return st;
  if (!qkv || !cos_t || !sin_t || !q_out || !table_len) return b200_fail(PAI_ERR_INVALID_ARG, "rope_append: NULL");
  if (((uintptr_t)qkv | (uintptr_t)q_out | (uintptr_t)cos_t | (uintptr_t)sin_t) & 15)
    return b200_fail(PAI_ERR_INVALID_ARG, "rope_append: qkv, q_out and the tables must be 16-byte aligned");
  p.h = (uint32_t)h, p.max_nodes = max_nodes, p.rows = rows, p.table_len = table_len;
  p.lens = lens, p.off = node_off, p.depth = depth, p.qkv = qkv, p.cos_t = cos_t, p.sin_t = sin_t, p.q = q_out;
  const CtxDeviceGuard on(ctx);
  if (on.status()) return on.status();
  const uint32_t per = kAppendThreads / (kv->head_dim / 8), heads = (uint32_t)h + 2 * kv->kv_heads;
  b200_launch(ctx, k_rope_append, dim3(max_nodes, kv->n_seq, (heads + per - 1) / per), dim3(kAppendThreads), 0, p);
  return b200_launched(ctx, 1, "k_rope_append");
}

extern "C" pai_status_t pai_b200_kv_accept_f16(pai_b200_ctx_t *ctx, const pai_b200_kv_view_t *kv, uint32_t max_path,
                                               const int32_t *lens, const int32_t *path, const int32_t *n_path,
                                               int32_t *lens_out) {
  KvDev c{};
  if (!ctx) return b200_fail(PAI_ERR_INVALID_ARG, "kv_accept: NULL context");
  pai_status_t st = kv_view_check(kv, "kv_accept", c);
  if (st) return st;
  if (!lens || !path || !n_path || !lens_out || !max_path) return b200_fail(PAI_ERR_INVALID_ARG, "kv_accept: NULL or empty");
  if (max_path > 1024) return b200_fail(PAI_ERR_UNSUPPORTED, "kv_accept: paths of %u (at most 1024)", max_path);
  const CtxDeviceGuard on(ctx);
  if (on.status()) return on.status();
  float *scratch;
  uint32_t *cnt;
  st = b200_ctx_scratch(ctx, 1, c.n_seq, &scratch, &cnt);
  if (st) return st;
  const uint32_t cols = c.hk * (c.hd / 8);
  b200_launch(ctx, k_kv_accept, dim3(2 * c.n_layer, (cols + kAcceptThreads - 1) / kAcceptThreads, c.n_seq),
              dim3(kAcceptThreads), max_path * 16, c, max_path, lens, path, n_path, lens_out, cnt);
  return b200_launched(ctx, 1, "k_kv_accept");
}

extern "C" pai_status_t pai_b200_kv_fork_f16(pai_b200_ctx_t *ctx, const pai_b200_kv_view_t *kv, uint32_t first,
                                             const int32_t *lens, const int32_t *parents, const int32_t *grow,
                                             int32_t *table_out, int32_t *lens_out, int32_t *granted) {
  ForkParams p{};
  if (!ctx) return b200_fail(PAI_ERR_INVALID_ARG, "kv_fork: NULL context");
  pai_status_t st = kv_view_check(kv, "kv_fork", p.c);
  if (st) return st;
  if (!lens || !lens_out || !granted) return b200_fail(PAI_ERR_INVALID_ARG, "kv_fork: NULL");
  const bool paged = kv->table != nullptr;
  const uint64_t entries = (uint64_t)kv->n_seq * kv->max_pages;
  if (paged && !table_out) return b200_fail(PAI_ERR_INVALID_ARG, "kv_fork: NULL table_out");
  if (paged && table_out < kv->table + entries && kv->table < table_out + entries)
    return b200_fail(PAI_ERR_INVALID_ARG, "kv_fork: table_out overlaps the table");
  if (!paged && kv->n_seq > 32)
    return b200_fail(PAI_ERR_UNSUPPORTED, "kv_fork: %u sequences without a page table (at most 32)", kv->n_seq);
  const CtxDeviceGuard on(ctx);
  if (on.status()) return on.status();
  p.first = first, p.paged = paged, p.lens = lens, p.parents = parents, p.grow = grow;
  p.table_out = table_out, p.lens_out = lens_out, p.granted = granted;
  // scratch: the copies (16 bytes each), then the pages' use, keepers and the free pages that are handed out
  const uint64_t words = 4ull * kv->n_seq + (paged ? 3ull * kv->n_pages : 0);
  float *scratch;
  uint32_t *cnt;
  st = b200_ctx_scratch(ctx, words, 1, &scratch, &cnt);
  if (st) return st;
  p.copies = (ForkCopy *)scratch;
  p.used = (int32_t *)(scratch + 4ull * kv->n_seq);
  p.keeper = p.used + kv->n_pages;
  p.fresh = p.keeper + kv->n_pages;
  b200_launch(ctx, k_kv_fork_plan, dim3(1), dim3(kPlanThreads), 0, p);
  // the copying kernel is resident before the plan is done, and waits for it
  const int pdl = b200_ctx_pdl(ctx);
  b200_ctx_set_pdl(ctx, 1);
  const uint32_t planes = 2 * kv->n_layer;
  if (paged) {
    const uint64_t pieces = (uint64_t)kv->page_tokens * (kv->head_dim / 8) * kv->kv_heads;
    const uint32_t z = (uint32_t)std::min<uint64_t>(
        64, std::max<uint64_t>(1, (pieces + kCopyThreads * kCopyBatch - 1) / (kCopyThreads * kCopyBatch)));
    b200_launch(ctx, k_kv_fork_pages, dim3(planes, kv->n_seq, z), dim3(kCopyThreads), 0, p.c, (const ForkCopy *)p.copies);
  } else {
    const uint64_t pieces = (uint64_t)kv->page_tokens * (kv->head_dim / 8);
    const uint32_t z = (uint32_t)std::min<uint64_t>(64, (pieces + kCopyThreads - 1) / kCopyThreads);
    const dim3 grid(planes, kv->kv_heads, z);
    if (kv->n_seq <= 8)
      b200_launch(ctx, k_kv_fork_runs<8>, grid, dim3(kCopyThreads), 0, p.c, (const ForkCopy *)p.copies);
    else
      b200_launch(ctx, k_kv_fork_runs<32>, grid, dim3(kCopyThreads), 0, p.c, (const ForkCopy *)p.copies);
  }
  b200_ctx_set_pdl(ctx, pdl);
  return b200_launched(ctx, 2, "k_kv_fork");
}
