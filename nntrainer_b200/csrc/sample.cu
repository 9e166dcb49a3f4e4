// SPDX-License-Identifier: Apache-2.0
/**
 * @file  sample.cu
 * @brief A token per row of logits, drawn with temperature, top-k, top-p and min-p from a random number that the caller gives.
 *
 * With w_i = exp((x_i - max x) / T) and the tokens in descending order of x, the lowest index first among equals: the first top_k of
 * them are kept, of these the shortest prefix whose weights reach top_p times their sum, of these those with w_i >= min_p. The token is
 * the first kept one, in ascending order of the index, up to which the kept weights exceed u times their sum.
 *
 * A token is right or wrong, so no rounding may decide it: weights are computed in double precision and kept as multiples of
 * 2^-44 in 64 bits, whose sums are exact in any order. What is left is where u * sum or top_p * sum falls within some 2^-44 of
 * a border.
 */
#include "common.cuh"

namespace nntr {

namespace {

constexpr int SP_THREADS = 512;
constexpr double SP_ONE = 17592186044416.0; // 2^44: 2^20 logits of the largest weight stay in 64 bits
constexpr unsigned SP_MAX_N = 1u << 20;

struct SampleArgs {
  const float *logits, *u, *row_params;
  long long ld;
  unsigned n;
  double temperature, top_p, min_p;
  unsigned top_k;
  unsigned *idx;
  float *idx_f, *prob;
};

/* bits that ascend with the value; 0 for what is never drawn: NaN and -inf */
__device__ __forceinline__ uint32_t order_of(float x) {
  if (!(x > -INFINITY))
    return 0u;
  const uint32_t b = __float_as_uint(x == 0.f ? 0.f : x); // -0 is 0
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}

struct Hist { // of a digit: how many, and the sum of their weights in two words
  uint32_t count[256], lo[256], hi[256];
};

__device__ __forceinline__ void hist_add(Hist &h, int digit, unsigned long long w) {
  atomicAdd(&h.count[digit], 1u);
  if (w) {
    const uint32_t add = (uint32_t)w, old = atomicAdd(&h.lo[digit], add);
    const uint32_t up = (uint32_t)(w >> 32) + (old + add < old); // the carry
    if (up)
      atomicAdd(&h.hi[digit], up);
  }
}

} // namespace

__global__ void __launch_bounds__(SP_THREADS) sample_kernel(SampleArgs a) {
  __shared__ Hist hist;
  __shared__ float s_max[SP_THREADS / 32];
  __shared__ uint32_t s_digit;
  __shared__ unsigned long long s_before, s_at;
  pdl_launch_dependents();
  pdl_wait();
  const int row = blockIdx.x, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const float *x = a.logits + row * a.ld;
  double temperature = a.temperature, top_p = a.top_p, min_p = a.min_p;
  unsigned top_k = a.top_k;
  if (a.row_params) {
    const float *p = a.row_params + 4ll * row;
    temperature = p[0], top_p = p[2], min_p = p[3];
    top_k = p[1] >= 1.f ? (unsigned)fminf(p[1], 1e9f) : 0u;
  }
  float mx = -INFINITY;
  for (unsigned i = tid; i < a.n; i += SP_THREADS)
    mx = fmaxf(mx, x[i]); // a NaN never wins
#pragma unroll
  for (int o = 16; o; o >>= 1)
    mx = fmaxf(mx, __shfl_xor_sync(FULL, mx, o));
  if (lane == 0)
    s_max[warp] = mx;
  __syncthreads();
  mx = s_max[0];
  for (int i = 1; i < SP_THREADS / 32; ++i)
    mx = fmaxf(mx, s_max[i]);
  if (mx == -INFINITY) { // nothing to draw from: the first token, as for the greatest of nothing
    if (tid == 0) {
      if (a.idx)
        a.idx[row] = 0;
      if (a.idx_f)
        a.idx_f[row] = 0.f;
      if (a.prob)
        a.prob[row] = 0.f;
    }
    return;
  }
  if (!(temperature > 0.0)) { // greedy
    temperature = 1.0;
    top_k = 1;
  }
  if (!(top_p > 0.0))
    top_k = 1;
  const double t = temperature, top = mx;
  auto weight_of = [&](float v) { return v == mx ? 1.0 : v > -INFINITY ? exp(((double)v - top) / t) : 0.0; };
  auto fixed_of = [&](float v) { return (unsigned long long)__double2ull_rn(weight_of(v) * SP_ONE); };

  /* The digit by digit search for the value (of `bits` bits) at which a running sum over the tokens reaches `target`: a sum of counts or of
   * weights, from the greatest value down or from the smallest up. Returns the value; *before: the sum in front of it, *at: the sum
   * (or count) of the tokens with that value. select(i, v, &key): whether token i takes part, and its value. */
  auto descend = [&](int bits, bool down, bool by_count, unsigned long long target, auto select, unsigned long long *before,
                     unsigned long long *at) {
    uint32_t prefix = 0;
    unsigned long long sum = 0;
    for (int shift = (bits - 1) / 8 * 8; shift >= 0; shift -= 8) {
      for (int i = tid; i < 256; i += SP_THREADS)
        hist.count[i] = hist.lo[i] = hist.hi[i] = 0;
      __syncthreads();
      for (unsigned i = tid; i < a.n; i += SP_THREADS) {
        const float v = x[i];
        uint32_t key;
        if (select(i, v, &key) && (unsigned long long)key >> (shift + 8) == prefix)
          hist_add(hist, (key >> shift) & 255, by_count ? 0ull : fixed_of(v));
      }
      __syncthreads();
      if (tid == 0) {
        unsigned long long run = sum;
        int d = down ? 255 : 0, last = -1;
        unsigned long long last_run = sum, last_at = 0;
        for (int k = 0; k < 256; ++k, d += down ? -1 : 1) {
          const unsigned long long here = by_count ? hist.count[d] : (unsigned long long)hist.hi[d] << 32 | hist.lo[d];
          if (here) {
            last = d, last_run = run, last_at = here;
            run += here;
            if (run >= target)
              break;
          }
        }
        s_digit = last < 0 ? 0 : last;
        s_before = last_run;
        s_at = last_at;
      }
      __syncthreads();
      prefix = prefix << 8 | s_digit;
      sum = s_before;
      *at = s_at;
      __syncthreads();
    }
    *before = sum;
    return prefix;
  };
  auto all = [&](unsigned, float v, uint32_t *key) { return (*key = order_of(v)) != 0; };

  // the cut: tokens above `cut` are kept, of those at it the ones with an index up to cut_idx
  uint32_t cut = 1;
  unsigned long long of_cut = ~0ull; // so many of those at the cut, the lowest indices
  unsigned long long before, at;
  bool have_cut = false;
  unsigned long long kept_sum = 0;
  if (top_k > 0 && top_k < a.n) {
    cut = descend(32, true, true, top_k, all, &before, &at);
    of_cut = top_k - before < at ? top_k - before : at; // all of them where there are fewer tokens than top_k
    have_cut = true;
  }
  auto weigh = [&](auto kept) { // exact in any order
    unsigned long long sum = 0;
    for (unsigned i = tid; i < a.n; i += SP_THREADS) {
      const float v = x[i];
      if (kept(i, v))
        sum += fixed_of(v);
    }
    if (tid == 0)
      s_at = 0;
    __syncthreads();
    atomicAdd(&s_at, sum);
    __syncthreads();
    sum = s_at;
    __syncthreads();
    return sum;
  };
  auto value_at = [&](uint32_t key) { // the value with these order bits
    return __uint_as_float(key & 0x80000000u ? key & 0x7fffffffu : ~key);
  };
  if (top_p > 0.0 && top_p < 1.0) {
    kept_sum = weigh([&](unsigned, float v) { return order_of(v) > (have_cut ? cut : 0u); });
    if (have_cut)
      kept_sum += of_cut * fixed_of(value_at(cut));
    const unsigned long long target = (unsigned long long)ceil(top_p * (double)kept_sum);
    const uint32_t c = descend(32, true, false, target, all, &before, &at);
    const unsigned long long w = fixed_of(value_at(c));
    unsigned long long r = target > before && w ? (target - before + w - 1) / w : 1;
    if (!have_cut || c > cut) {
      cut = c, of_cut = r, have_cut = true;
    } else if (c == cut && r < of_cut) {
      of_cut = r;
    }
  }
  uint32_t cut_idx = 0xffffffffu;
  if (have_cut) { // the of_cut-th token at the cut
    auto equal = [&](unsigned i, float v, uint32_t *key) {
      *key = i;
      return order_of(v) == cut;
    };
    cut_idx = descend(20, false, true, of_cut, equal, &before, &at);
  }
  auto kept = [&](unsigned i, float v) {
    const uint32_t o = order_of(v);
    return o && (!have_cut || o > cut || (o == cut && i <= cut_idx)) && (v == mx || weight_of(v) >= min_p);
  };
  const unsigned long long total = weigh(kept);
  const double u = a.u[row];
  unsigned long long target = u > 0.0 ? (unsigned long long)fmin(u * (double)total, (double)total) + 1 : 1; // the first sum above u * total
  if (target > total)
    target = total;
  const uint32_t id = descend(20, false, false, target, [&](unsigned i, float v, uint32_t *key) { *key = i; return kept(i, v); }, &before, &at);
  if (tid == 0) {
    if (a.idx)
      a.idx[row] = id;
    if (a.idx_f)
      a.idx_f[row] = (float)id;
    if (a.prob)
      a.prob[row] = (float)(weight_of(x[id]) * SP_ONE / (double)total);
  }
}

int launch_sample(const float *logits, int64_t rows, int64_t n, int64_t ld, const float *u, double temperature, unsigned top_k, double top_p,
                  double min_p, const float *row_params, unsigned *idx, float *idx_f, float *prob, unsigned flags, cudaStream_t st) {
  if (rows == 0)
    return NNTR_CUDA_OK;
  if (!logits || !u || (!idx && !idx_f) || rows < 0 || n <= 0 || (rows > 1 && ld < n))
    return set_error(NNTR_CUDA_ERR_INVALID, "sample: bad arguments (%lld rows of %lld logits, %lld apart)", (long long)rows, (long long)n,
                     (long long)ld);
  if (n > SP_MAX_N || rows > 65535)
    return set_error(NNTR_CUDA_ERR_UNSUPPORTED, "sample: at most 65535 rows of at most %u logits", SP_MAX_N);
  if (!row_params && (!(temperature >= 0.0) || !(top_p >= 0.0) || !(min_p >= 0.0 && min_p <= 1.0)))
    return set_error(NNTR_CUDA_ERR_INVALID, "sample: temperature %g, top_p %g, min_p %g; need temperature and top_p >= 0, min_p from 0 to 1",
                     temperature, top_p, min_p);
  SampleArgs a = {logits, u, row_params, ld, (unsigned)n, temperature, top_p, min_p, top_k, idx, idx_f, prob};
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = (flags & NNTR_CUDA_GEMV_PDL) ? 1 : 0;
  cfg.stream = st;
  cfg.gridDim = dim3((unsigned)rows);
  cfg.blockDim = dim3(SP_THREADS);
  const cudaError_t e = cudaLaunchKernelEx(&cfg, sample_kernel, a);
  count_launch();
  return check_cuda(e, "sample launch");
}

} // namespace nntr
