// SPDX-License-Identifier: Apache-2.0
/**
 * @file  paged_attention.cuh
 * @brief What the attention kernels over a cache in pages share: arguments, which cache rows a tile of queries sees, the
 *        exponential.
 */
#ifndef NNTR_PAGED_ATTENTION_CUH_
#define NNTR_PAGED_ATTENTION_CUH_

#include "paged.cuh"

namespace nntr {

struct AttendArgs {
  const void *q, *k, *v;
  void *out;
  const float *sink;
  long long ld_q, ld_out;
  int window, first; // window: INT_MAX / 2 where there is none
  int out_f32;
  float scale_log2; // log2(e) / sqrt(head_dim)
};

/** 2^x, the hardware's approximation (2^-22) */
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

constexpr float LOG2E = 1.4426950408889634f;
/** log2 of what a row's greatest probability is when its maximum is taken */
constexpr float PAGED_LIFT = 6.f;

/* Blocks of KEYS cache rows that hold what a tile of queries at positions lo .. hi sees: those of the first tokens, then the window's.
 * A row in none of the queries' sight counts as not there: it may hold anything. */
struct Sight {
  int lo, hi, window, first, from, head_blocks, first_block, blocks;
  __device__ __forceinline__ Sight(int lo_, int hi_, int window_, int first_, int keys) : lo(lo_), hi(hi_), window(window_) {
    from = max(0, lo - window + 1);
    first = min(first_, from);
    head_blocks = (first + keys - 1) / keys;
    first_block = from / keys;
    if (first_block <= head_blocks)
      head_blocks = first_block = 0;
    blocks = hi < 0 ? 0 : head_blocks + hi / keys - first_block + 1;
  }
  __device__ __forceinline__ int block(int i) const { return i < head_blocks ? i : i - head_blocks + first_block; }
  __device__ __forceinline__ bool row_read(int j) const { return j <= hi && (j >= from || j < first); } // by one query at least
};

/* chunks of queries (paged_attention_chunk.cu) */
int launch_paged_attention_chunk(const AttendArgs &a, int dtype, const PagedGeom &g, const PagedBatch &s, unsigned max_rows, unsigned flags,
                                 cudaStream_t st);

} // namespace nntr
#endif
