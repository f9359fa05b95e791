// The paged key/value cache as its kernels see it: checks of the C ABI's
// structs, sequence look-up and slot addresses.
#pragma once

#include "internal.h"
#include "ptx.cuh"

namespace ncm {

// Sequences of one call, resolved on the device (ncm_kv_batch_t).
struct KvBatch {
  const int32_t* token_start;
  const int32_t* kv_lens;
  const int32_t* page_table;
  long long table_stride;
  int table_width;
  int batch;
  long long rows;
};

struct KvPools {
  void* k;
  void* v;
  float* k_scale;
  float* v_scale;
  int kv_heads;
  int page_shift;  // log2 of the page size
  int num_pages;
};

inline KvBatch kv_batch_of(const ncm_kv_batch_t* b) {
  return KvBatch{b->token_start, b->kv_lens, b->page_table, b->table_stride, b->table_width, b->batch, b->rows};
}

inline KvPools kv_pools_of(const ncm_kv_cache_t* c) {
  int shift = 0;
  while ((1 << shift) < c->page_size) ++shift;
  return KvPools{c->k, c->v, c->k_scale, c->v_scale, c->kv_heads, shift, static_cast<int>(c->num_pages)};
}

inline int kv_check_cache(const char* what, const ncm_kv_cache_t* c) {
  if (c == nullptr) return ncm_fail(NCM_EINVAL, "%s: null cache", what);
  if (c->format < NCM_KV_BF16 || c->format > NCM_KV_E4M3) return ncm_fail(NCM_EINVAL, "%s: bad format %d", what, c->format);
  if (c->head_dim != 64 && c->head_dim != 128)
    return ncm_fail(NCM_EINVAL, "%s: head_dim %d must be 64 or 128", what, c->head_dim);
  if (c->page_size < 8 || c->page_size > 1024 || (c->page_size & (c->page_size - 1)) != 0)
    return ncm_fail(NCM_EINVAL, "%s: page_size %d must be a power of two from 8 to 1024", what, c->page_size);
  if (c->kv_heads < 1 || c->kv_heads > 1024 || c->num_pages < 1 ||
      c->num_pages > INT32_MAX / (static_cast<int64_t>(c->kv_heads) * c->page_size))
    return ncm_fail(NCM_EINVAL, "%s: bad pool shape (%lld pages, %d heads)", what, (long long)c->num_pages, c->kv_heads);
  if (!c->k || !c->v || !aligned_to(c->k, 16) || !aligned_to(c->v, 16))
    return ncm_fail(NCM_EINVAL, "%s: the pools must be 16-byte aligned buffers", what);
  if (c->format != NCM_KV_BF16 && (!c->k_scale || !c->v_scale || !aligned_to(c->k_scale, 4) || !aligned_to(c->v_scale, 4)))
    return ncm_fail(NCM_EINVAL, "%s: a quantised cache needs its scales", what);
  return NCM_OK;
}

inline int kv_check_batch(const char* what, const ncm_kv_batch_t* b, bool need_lens) {
  if (b == nullptr) return ncm_fail(NCM_EINVAL, "%s: null batch", what);
  if (b->batch < 0 || b->rows < 0 || b->rows > INT32_MAX || b->table_width < 0 || b->table_stride < b->table_width ||
      b->table_stride > INT64_MAX / 8 / (static_cast<int64_t>(b->batch) + 1))
    return ncm_fail(NCM_EINVAL, "%s: bad batch (batch=%d rows=%lld table %d of %lld)", what, b->batch,
                    (long long)b->rows, b->table_width, (long long)b->table_stride);
  if (b->batch == 0) return NCM_OK;
  if (!b->token_start || (need_lens && !b->kv_lens) || (b->table_width > 0 && !b->page_table))
    return ncm_fail(NCM_EINVAL, "%s: null batch array", what);
  if (!aligned_to(b->token_start, 4) || !aligned_to(b->kv_lens, 4) || !aligned_to(b->page_table, 4))
    return ncm_fail(NCM_EINVAL, "%s: misaligned batch array", what);
  return NCM_OK;
}

// A [rows, width] bf16 row array of the caller's.
inline int kv_check_rows(const char* what, const char* name, const void* p, int64_t stride, int64_t rows, int64_t width) {
  if (stride < width || stride % 8 != 0 || stride > INT64_MAX / 8 / (rows + 1))
    return ncm_fail(NCM_EINVAL, "%s: row stride %lld of %s must be a multiple of 8 and cover %lld columns", what,
                    (long long)stride, name, (long long)width);
  if (rows > 0 && (p == nullptr || !aligned_to(p, 16)))
    return ncm_fail(NCM_EINVAL, "%s: %s must be a 16-byte aligned buffer", what, name);
  return NCM_OK;
}

// The sequence that owns packed row t: the b with token_start[b] <= t <
// token_start[b + 1], or -1. Bounds that do not ascend can only give a wrong b
// in range, whose own bounds the caller checks.
__device__ __forceinline__ int sequence_of_row(const int32_t* token_start, int batch, long long t) {
  int lo = 0, n = batch;  // the answer is in [lo, lo + n)
  while (n > 1) {
    const int half = n >> 1;
    if (__ldg(token_start + lo + half) <= t) {
      lo += half;
      n -= half;
    } else {
      n = half;
    }
  }
  if (batch < 1 || __ldg(token_start + lo) > t || __ldg(token_start + lo + 1) <= t) return -1;
  return lo;
}

// Keys that a sequence has at most: what its row of the page table covers, and
// 2^30, so that a position plus a tile stays in 32 bits.
__device__ __forceinline__ int kv_capacity(const KvBatch& b, const KvPools& c) {
  return static_cast<int>(min(static_cast<long long>(b.table_width) << c.page_shift, 1ll << 30));
}

// Element offset of slot `off` of page `page`, head `h`, in units of rows.
__device__ __forceinline__ long long kv_slot(const KvPools& c, int page, int h, int off) {
  return ((static_cast<long long>(page) * c.kv_heads + h) << c.page_shift) + off;
}

}  // namespace ncm
