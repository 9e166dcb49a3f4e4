// SPDX-License-Identifier: Apache-2.0
/**
 * @file  paged.cuh
 * @brief A key/value cache in pages and a batch of sequences on it, as the kernels see them: argument checks, the way from
 *        a row of a sequence to its address, the conversions of 16-bit values.
 */
#ifndef NNTR_PAGED_CUH_
#define NNTR_PAGED_CUH_

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.cuh"

namespace nntr {

/** nntr_paged_batch on the device side. Nothing in the arrays is trusted: see seq_rows() and row_offset(). */
struct PagedBatch {
  const int *row_start, *context, *table;
  int batch, tokens, max_new, ld_table, table_rows; // table_rows: cache rows that a sequence's entries of the table stand for
};
struct PagedGeom {
  long long page_stride; // elements
  int page_shift, n_pages, hq, hkv, hd;

  /** Element offset of row `row` of kv head h in sequence b, or -1 where the page table names no page of the pool. 64 bits: a
   *  pool passes 2^31 elements early. */
  __device__ __forceinline__ long long row_offset(const PagedBatch &s, int b, int row, int h) const {
    const int slot = row >> page_shift;
    if (row < 0 || slot >= s.ld_table)
      return -1;
    const int page = __ldg(s.table + (size_t)b * s.ld_table + slot);
    if ((unsigned)page >= (unsigned)n_pages)
      return -1;
    return page * page_stride + ((long long)(row & ((1 << page_shift) - 1)) * hkv + h) * hd;
  }
};

/** A sequence's query rows [first, first + n) and the position of the first one; bad: the arrays contradict themselves or the
 *  bounds that came with them. Then no row outside q is in it, and no more than max_new. A negative position sees nothing. Whatever the
 *  arrays hold, -tokens <= pos and pos + n <= table_rows: a row up to a query's position that is not negative has an entry in the page table. */
struct SeqRows {
  int first, n, pos;
  bool bad;
};
__device__ __forceinline__ SeqRows seq_rows(const PagedBatch &s, int lo, int hi, int given) { // row_start of it and of the next one, context
  const int ctx = max(0, min(given, s.table_rows)); // from both sides: the difference below stays in 32 bits
  SeqRows r;
  r.first = min(max(lo, 0), s.tokens);
  const int end = min(max(hi, r.first), s.tokens);
  r.n = min(end - r.first, s.max_new);
  r.pos = ctx - (end - r.first);
  r.bad = lo < 0 || hi < lo || hi > s.tokens || hi - lo > s.max_new || r.pos < 0 || given != ctx;
  return r;
}
__device__ __forceinline__ SeqRows seq_rows(const PagedBatch &s, int b) {
  return seq_rows(s, __ldg(s.row_start + b), __ldg(s.row_start + b + 1), __ldg(s.context + b));
}
/** The sequence that query row `token` belongs to, by all lanes of a warp; batch where it lies behind the last one. */
__device__ __forceinline__ int seq_of_row(const PagedBatch &s, int token, int lane) {
  int seq = 0;
  for (int b0 = 0; b0 < s.batch; b0 += 32) { // row_start ascends: as many sequences end at or in front of the row as lie in front of it
    const int b = b0 + lane;
    const unsigned m = __ballot_sync(FULL, b < s.batch && __ldg(s.row_start + b + 1) <= token);
    seq += __popc(m);
    if (m != FULL)
      break;
  }
  return seq;
}

/* two values to 16 bits, to nearest; one word */
template <typename T> __device__ __forceinline__ uint32_t pack2(float a, float b);
template <> __device__ __forceinline__ uint32_t pack2<__half>(float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t *>(&h);
}
template <> __device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float a, float b) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t *>(&h);
}
__device__ __forceinline__ float widen(__half h) { return __half2float(h); }
__device__ __forceinline__ float widen(__nv_bfloat16 h) { return __bfloat162float(h); }

/** Checks of what every paged call is given (host); fills the device-side forms. */
int check_paged(const char *what, const nntr_paged_cache *c, const nntr_paged_batch *b, PagedGeom *g, PagedBatch *s);

} // namespace nntr
#endif
