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
/* What a row's probabilities may be. The greatest is 2^LIFT when the maximum is taken that they refer to; the rows behind go by that maximum
 * while no thread's sum of a step (a lane's four, or half a row of a step) is above MOST, so that each probability fits its type, and beyond it
 * the step begins again. So a row's greatest probability lies between 2^LIFT and MOST, and so does the exponent that a sink meets. fp16: the small
 * ones of a long context stay out of the subnormal numbers. bf16 has the exponents of fp32: probabilities of at most 1 leave those to the
 * values, whose sums overflow only where rows * |value| does. FROM .. UPTO: exponents x of 2^x that the polynomial of
 * paged_attention_chunk.cu tells apart; what is further down is as nothing beside 2^LIFT, what is further up, and a NaN, counts as UPTO, which is
 * above MOST. */
template <typename T> struct Weights;
template <> struct Weights<__half> {
  static constexpr float LIFT = 6.f, MOST = 32768.f, FROM = -48.f, UPTO = 16.f; // 2^-48: zero in fp16
};
template <> struct Weights<__nv_bfloat16> {
  static constexpr float LIFT = -9.f, MOST = 1.f, FROM = -127.f, UPTO = 1.f;
};

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
  __device__ __forceinline__ bool any_read(int j, int n) const { return j <= hi && (j + n > from || j < first); } // of the rows j .. j + n - 1
};

/* chunks of queries (paged_attention_chunk.cu) */
int launch_paged_attention_chunk(const AttendArgs &a, int dtype, const PagedGeom &g, const PagedBatch &s, unsigned max_rows, unsigned flags,
                                 cudaStream_t st);

} // namespace nntr
#endif
