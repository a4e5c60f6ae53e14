// The fp16 cache view of pai_b200_kv_view_t on the device, and the checks
// its entry points share.
#pragma once
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "../b200_internal.h"

struct KvDev {
  __half *k, *v;         // one layer's planes, or all layers' with layer_stride
  const int32_t *table;  // [n_seq][max_pages], NULL: page s
  uint32_t n_layer, n_seq, hk, hd, page_tokens, n_pages, max_pages;
  uint64_t layer_stride, page_stride, head_stride;
};

// Element offset of row `pos` of sequence s (layer 0, kv head 0), or -1 for a
// hole or a position behind the last page.
__host__ __device__ __forceinline__ int64_t kv_row(const KvDev &c, uint32_t s, uint32_t pos) {
  const uint32_t pg = pos / c.page_tokens;
  if (pg >= c.max_pages) return -1;
  const uint32_t page = c.table ? (uint32_t)c.table[(size_t)s * c.max_pages + pg] : s;
  if (page >= c.n_pages) return -1;
  return (int64_t)(page * c.page_stride + (uint64_t)(pos - pg * c.page_tokens) * c.hd);
}

// Committed positions of sequence s: lens[s] within [0, max_pages * page_tokens].
__host__ __device__ __forceinline__ uint32_t kv_len(const KvDev &c, const int32_t *lens, uint32_t s) {
  const int32_t n = lens[s];
  const uint32_t cap = c.max_pages * c.page_tokens;
  return n < 0 ? 0u : (uint32_t)n < cap ? (uint32_t)n : cap;
}

// First row and node count of sequence s, within the `rows` rows and max_nodes.
__host__ __device__ __forceinline__ uint32_t kv_nodes(const int32_t *off, uint32_t s, uint64_t rows, uint32_t max_nodes,
                                             uint32_t *first) {
  const int64_t a = off[s], b = off[s + 1];
  *first = 0;
  if (a < 0 || b <= a || (uint64_t)a >= rows) return 0;
  *first = (uint32_t)a;
  const uint64_t n = (uint64_t)(b - a), left = rows - (uint64_t)a;
  return (uint32_t)(n < left ? (n < max_nodes ? n : max_nodes) : (left < max_nodes ? left : max_nodes));
}

// The rules of pai_b200_kv_view_t, and its device form.
static inline pai_status_t kv_view_check(const pai_b200_kv_view_t *kv, const char *op, KvDev &c) {
  if (!kv || !kv->k || !kv->v) return b200_fail(PAI_ERR_INVALID_ARG, "%s: NULL cache", op);
  if (((uintptr_t)kv->k | (uintptr_t)kv->v) & 15)
    return b200_fail(PAI_ERR_INVALID_ARG, "%s: K/V planes must be 16-byte aligned", op);
  if (!kv->n_layer || !kv->n_seq || !kv->kv_heads || !kv->head_dim || !kv->page_tokens || !kv->n_pages || !kv->max_pages)
    return b200_fail(PAI_ERR_INVALID_ARG, "%s: a cache size is 0", op);
  if ((kv->layer_stride | kv->page_stride | kv->head_stride) & 7)
    return b200_fail(PAI_ERR_INVALID_ARG, "%s: cache strides must be multiples of 8 elements", op);
  if ((uint64_t)kv->max_pages * kv->page_tokens > 0x7FFFFFFFull)
    return b200_fail(PAI_ERR_INVALID_ARG, "%s: %u pages of %u positions", op, kv->max_pages, kv->page_tokens);
  if ((uint64_t)kv->max_pages * kv->n_seq > 0x7FFFFFFFull)
    return b200_fail(PAI_ERR_UNSUPPORTED, "%s: a table of %u x %u pages", op, kv->n_seq, kv->max_pages);
  if (kv->n_pages > 0x7FFFFFFFu) return b200_fail(PAI_ERR_INVALID_ARG, "%s: %u pages", op, kv->n_pages);
  if (!kv->table && (kv->max_pages != 1 || kv->n_pages < kv->n_seq))
    return b200_fail(PAI_ERR_INVALID_ARG, "%s: a cache without a table has one page for each sequence", op);
  if (kv->head_stride < (uint64_t)kv->page_tokens * kv->head_dim && kv->kv_heads > 1)
    return b200_fail(PAI_ERR_MISMATCH, "%s: head stride %llu below %u positions of %u", op,
                     (unsigned long long)kv->head_stride, kv->page_tokens, kv->head_dim);
  if (kv->head_dim % 8 || kv->head_dim > 256)
    return b200_fail(PAI_ERR_UNSUPPORTED, "%s: head_dim %u (a multiple of 8 up to 256)", op, kv->head_dim);
  if (kv->n_seq > 1024 || kv->kv_heads > 1024 || kv->n_layer > 65535)
    return b200_fail(PAI_ERR_UNSUPPORTED, "%s: %u sequences, %u kv heads, %u layers", op, kv->n_seq, kv->kv_heads,
                     kv->n_layer);
  c.k = (__half *)kv->k, c.v = (__half *)kv->v, c.table = kv->table;
  c.n_layer = kv->n_layer, c.n_seq = kv->n_seq, c.hk = kv->kv_heads, c.hd = kv->head_dim;
  c.page_tokens = kv->page_tokens, c.n_pages = kv->n_pages, c.max_pages = kv->max_pages;
  c.layer_stride = kv->layer_stride, c.page_stride = kv->page_stride, c.head_stride = kv->head_stride;
  return PAI_OK;
}

// The shared rules of the operators on drafted nodes; `c` becomes the view of one layer.
static inline pai_status_t kv_nodes_check(const pai_b200_kv_view_t *kv, const char *op, uint32_t layer, uint64_t h,
                                          uint64_t rows, uint32_t max_nodes, const int32_t *lens,
                                          const int32_t *node_off, KvDev &c) {
  pai_status_t st = kv_view_check(kv, op, c);
  if (st) return st;
  if (!lens || !node_off) return b200_fail(PAI_ERR_INVALID_ARG, "%s: NULL lengths", op);
  if (layer >= kv->n_layer) return b200_fail(PAI_ERR_INVALID_ARG, "%s: layer %u of %u", op, layer, kv->n_layer);
  if (h == 0 || h % kv->kv_heads || h > 4096)
    return b200_fail(PAI_ERR_INVALID_ARG, "%s: heads %llu / kv heads %u", op, (unsigned long long)h, kv->kv_heads);
  if (rows == 0 || rows > 0x7FFFFFFFull || max_nodes == 0)
    return b200_fail(PAI_ERR_INVALID_ARG, "%s: %llu rows, at most %u nodes", op, (unsigned long long)rows, max_nodes);
  if (max_nodes > 1024) return b200_fail(PAI_ERR_UNSUPPORTED, "%s: %u nodes of a sequence (at most 1024)", op, max_nodes);
  c.k += (size_t)layer * c.layer_stride;
  c.v += (size_t)layer * c.layer_stride;
  return PAI_OK;
}
