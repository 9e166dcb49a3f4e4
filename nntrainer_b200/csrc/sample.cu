// SPDX-License-Identifier: Apache-2.0
/**
 * @file  sample.cu
 * @brief A token per row of logits, drawn with temperature, top-k, top-p and min-p from a random number that the caller gives.
 *
 * With w_i = exp((x_i - max x) / T) and the tokens in descending order of x, the lowest index first among equals: the first top_k of
 * them are kept, of these the shortest prefix whose weights reach top_p times their sum, of these those with w_i >= min_p. The token is
 * the first kept one, in ascending order of the index, up to which the kept weights exceed u times their sum.
 *
 * A token is right or wrong, so the sums must not depend on their order: weights are whole multiples of 2^-44 in 64 bits. The ones that
 * count most (a few thousand of the greatest logits, down to 2^-14 of the greatest weight) are computed in double precision, the rest
 * of the row in fp32 to 2^-22 of themselves.
 *
 * A row is read for its greatest logit, an eighth of it for a histogram that says from which value up there are about SP_HEAD logits, and
 * again (from L2) for the list of these and the sum of the others. The first CTA of the row's cluster holds the list in shared memory and finds
 * the cuts and the draw by digits of eight bits, each a histogram. Where a cut lies below the list, the histogram says
 * about where; one more pass lists the logits around it and sums what is above, slice by slice. Where that does not do either (very many
 * equal logits, top_k and top_p both far down) the whole cluster goes by digits over the whole row.
 */
#include "cluster.cuh"
#include "pipeline.cuh"

#include <algorithm>
#include <atomic>

namespace nntr {

namespace {

constexpr int SP_THREADS = 512, SP_WARPS = SP_THREADS / 32;
constexpr int SP_MAX_PARTS = 8;
constexpr int SP_LIST = 12288;             // logits that the list holds
constexpr int SP_HEAD = 4096;              // logits that it is meant for, the greatest ones
constexpr int SP_AROUND = 8000;            // ... and around a cut further down: three standard deviations of the estimate and more
constexpr int SP_BINS = 512;               // of the estimate, over 46 powers of two of the weight
constexpr int SP_EVERY = 8;                // every eighth block of 128 logits is in it
constexpr double SP_ONE = 17592186044416.0; // 2^44: 2^20 logits of the greatest weight stay in 64 bits
constexpr double SP_EXACT_NATS = 9.7;      // (x - max) / T of the lightest token in double precision: 2^-14
constexpr unsigned SP_MAX_N = 1u << 20;

struct SampleArgs {
  const float *logits, *u, *row_params;
  long long ld;
  unsigned n, sub_len; // sub_len: logits of a warp's slice
  int vec;             // rows are 16-byte aligned
  double temperature, top_p, min_p;
  unsigned top_k;
  unsigned *idx;
  float *idx_f, *prob;
};

struct SampleShared {
  float x[SP_LIST];
  uint32_t i[SP_LIST];
  uint32_t hist[2][2][256]; // of a digit: the sum of its tokens' weights in two words
  uint32_t bins[SP_BINS], all_bins[SP_BINS]; // of this CTA's part of the row, of the row
  unsigned long long sub[SP_MAX_PARTS * SP_WARPS], sum[SP_WARPS], before, at;
  float max_of[SP_MAX_PARTS], warp_max[SP_WARPS], min_x, from, upto;
  uint32_t counts[SP_MAX_PARTS], above[SP_MAX_PARTS], count, n_above, digit, verdict;
};

/* bits that ascend with the value; 0 for what is never drawn: NaN and -inf */
__device__ __forceinline__ uint32_t order_of(float x) {
  if (!(x > -INFINITY))
    return 0u;
  const uint32_t b = __float_as_uint(x == 0.f ? 0.f : x); // -0 is 0
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float value_of(uint32_t order) { return __uint_as_float(order & 0x80000000u ? order & 0x7fffffffu : ~order); }

/* Weights of a row. 2^f on [-1/2, 1/2]: polynomial of the least greatest relative error (2^-28.9) with value 1 at 0. */
struct Weigher {
  float mx, exact_from; // the greatest logit; from here up in double precision
  double top, per_t;
  float c_hi, c_lo; // log2(e) / T

  __device__ __forceinline__ Weigher(float mx_, double t) : mx(mx_), top(mx_), per_t(1.0 / t) {
    exact_from = fmaxf((float)(top - SP_EXACT_NATS * t), -3.402823466e38f);
    const double c = 1.4426950408889634 / t;
    c_hi = (float)c;
    c_lo = isinf(c_hi) ? 0.f : (float)(c - (double)c_hi);
  }
  __device__ __forceinline__ double exactly(float x) const { return x == mx ? 1.0 : x > -INFINITY ? exp(((double)x - top) * per_t) : 0.0; }
  __device__ __forceinline__ unsigned long long in_fp32(float x) const {
    const float d = x - mx;
    const float e = fabsf(x) > fabsf(mx) ? (x - d) - mx : x - (d + mx); // what the difference was rounded by
    const float y = d * c_hi;
    if (!(y > -46.f))
      return 0ull;
    const float n = rintf(y), f = fmaf(d, c_hi, -n) + fmaf(d, c_lo, e * c_hi);
    float q = 1.535336190840639e-4f;
    q = fmaf(q, f, 1.3398874413974103e-3f);
    q = fmaf(q, f, 9.618437357669995e-3f);
    q = fmaf(q, f, 5.550332471126199e-2f);
    q = fmaf(q, f, 2.4022647913628897e-1f);
    q = fmaf(q, f, 6.931472028550653e-1f);
    return (unsigned long long)__float2uint_rn(fmaf(q, f, 1.f) * 1073741824.f) << 14 >> (int)-n;
  }
  __device__ __forceinline__ unsigned long long operator()(float x) const {
    return x >= exact_from ? __double2ull_rn(exactly(x) * SP_ONE) : in_fp32(x);
  }
  /* the least logit with a weight of at least w, but no greater than the greatest */
  __device__ float least_with(double w) const {
    float v = (float)(top + log(w) / per_t);
    if (!(v < mx))
      return mx;
    for (int k = 0; k < 8 && v > -3e38f && exactly(nextafterf(v, -INFINITY)) >= w; ++k)
      v = nextafterf(v, -INFINITY);
    for (int k = 0; k < 8 && v < mx && exactly(v) < w; ++k)
      v = nextafterf(v, INFINITY);
    return v;
  }
};

__device__ __forceinline__ void st_remote32(void *mine, int rank, uint32_t v) {
  uint32_t remote;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(smem_u32(mine)), "r"(rank));
  asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(remote), "r"(v) : "memory");
}
__device__ __forceinline__ void st_remote64(void *mine, int rank, unsigned long long v) {
  uint32_t remote;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(smem_u32(mine)), "r"(rank));
  asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(remote), "l"(v) : "memory");
}
__device__ __forceinline__ uint32_t ld_remote32(const void *mine, int rank) {
  uint32_t remote, v;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(smem_u32(mine)), "r"(rank));
  asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(remote) : "memory");
  return v;
}
__device__ __forceinline__ unsigned long long warp_scan(unsigned long long v, int lane) { // sums up to and with the lane's
#pragma unroll
  for (int o = 1; o < 32; o *= 2) {
    const unsigned long long t = __shfl_up_sync(FULL, v, o);
    v += lane >= o ? t : 0;
  }
  return v;
}
__device__ __forceinline__ unsigned long long warp_sum(unsigned long long v) {
#pragma unroll
  for (int o = 16; o; o >>= 1)
    v += __shfl_xor_sync(FULL, v, o);
  return v;
}

/* Sum over the CTA, in every thread. */
__device__ unsigned long long cta_sum(SampleShared &sh, unsigned long long v) {
  v = warp_sum(v);
  __syncthreads();
  if ((threadIdx.x & 31) == 0)
    sh.sum[threadIdx.x >> 5] = v;
  __syncthreads();
  v = 0;
  for (int i = 0; i < SP_WARPS; ++i)
    v += sh.sum[i];
  return v;
}

/* Digit by digit search for the value (of `bits` bits) at which a running sum over tokens reaches `target` (or ends, if it does not), from the
 * greatest value down or from the smallest up. each(f) calls f(value, weight) for this CTA's tokens, weight 1 to count them; parts:
 * CTAs that take part. *before: the sum in front of the value, *at: that of its tokens. */
template <class Each>
__device__ uint32_t descend(SampleShared &sh, int parts, int bits, bool down, unsigned long long target, Each each,
                            unsigned long long *before, unsigned long long *at) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  uint32_t prefix = 0;
  unsigned long long sum = 0;
  *at = 0;
  int side = 0;
  for (int shift = (bits - 1) / 8 * 8; shift >= 0; shift -= 8, side ^= 1) {
    auto &h = sh.hist[side];
    for (int i = tid; i < 2 * 256; i += SP_THREADS)
      h[i >> 8][i & 255] = 0;
    __syncthreads();
    each([&](uint32_t key, unsigned long long w) {
      if ((unsigned long long)key >> (shift + 8) == prefix && w) {
        const int d = key >> shift & 255;
        const uint32_t add = (uint32_t)w, old = atomicAdd(&h[0][d], add), up = (uint32_t)(w >> 32) + (old + add < old);
        if (up) // with the carry
          atomicAdd(&h[1][d], up);
      }
    });
    if (parts > 1) { // the next level uses the other histogram: nobody writes into this one while it is read
      cluster_sync();
      unsigned long long all = 0;
      if (tid < 256)
        for (int k = 0; k < parts; ++k)
          all += (unsigned long long)ld_remote32(&h[1][tid], k) << 32 | ld_remote32(&h[0][tid], k);
      cluster_sync();
      if (tid < 256) {
        h[0][tid] = (uint32_t)all;
        h[1][tid] = (uint32_t)(all >> 32);
      }
    }
    __syncthreads();
    if (warp == 0) {
      unsigned long long v[8], run = 0;
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const int d = down ? 255 - (8 * lane + k) : 8 * lane + k;
        v[k] = (unsigned long long)h[1][d] << 32 | h[0][d];
        run += v[k];
      }
      const unsigned long long upto = warp_scan(run, lane) + sum, all = __shfl_sync(FULL, upto, 31);
      const unsigned long long goal = target < all ? target : all;
      const unsigned m = __ballot_sync(FULL, run > 0 && upto >= goal);
      if (m == 0 ? lane == 0 : lane == __ffs(m) - 1) {
        unsigned long long in_front = upto - run;
        int k = 0;
        while (k < 7 && !(v[k] && in_front + v[k] >= goal))
          in_front += v[k++];
        sh.digit = down ? 255 - (8 * lane + k) : 8 * lane + k;
        sh.before = in_front;
        sh.at = v[k];
      }
    }
    __syncthreads();
    prefix = prefix << 8 | sh.digit;
    sum = sh.before;
    *at = sh.at;
  }
  *before = sum;
  __syncthreads();
  return prefix;
}

} // namespace

__global__ void __launch_bounds__(SP_THREADS) sample_kernel(SampleArgs a) {
  extern __shared__ __align__(16) uint8_t smem[];
  SampleShared &sh = *reinterpret_cast<SampleShared *>(smem);
  pdl_launch_dependents();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int parts = cluster_size(), part = cluster_rank(), row = blockIdx.x / parts;
  if (parts > 1)
    cluster_arrive(); // every CTA has started before one writes into another
  pdl_wait();
  const float *x = a.logits + row * a.ld;
  double temperature = a.temperature, top_p = a.top_p, min_p = a.min_p;
  unsigned top_k = a.top_k;
  if (a.row_params) {
    const float *p = a.row_params + 4ll * row;
    temperature = p[0] <= 1e30f ? p[0] : p[0] > 0.f ? 1e30f : 0.f, top_p = p[2], min_p = p[3];
    top_k = p[1] >= 1.f ? (unsigned)fminf(p[1], 1e9f) : 0u;
  }
  // this warp's slice of the row
  const unsigned s0 = min(a.n, (unsigned)(part * SP_WARPS + warp) * a.sub_len), s1 = min(a.n, s0 + a.sub_len);
  constexpr int AT = 4; // loads of a lane on their way at a time
  auto for_slice = [&](auto f) { // f(index, four logits); what is behind the slice is NaN
    for (unsigned i0 = s0 + 4 * lane; i0 - 4 * lane < s1; i0 += 128 * AT) {
      float4 v[AT];
#pragma unroll
      for (int k = 0; k < AT; ++k) {
        const unsigned i = i0 + 128 * k;
        if (a.vec && i + 4 <= s1)
          v[k] = *reinterpret_cast<const float4 *>(x + i);
        else
          v[k] = make_float4(i < s1 ? x[i] : NAN, i + 1 < s1 ? x[i + 1] : NAN, i + 2 < s1 ? x[i + 2] : NAN, i + 3 < s1 ? x[i + 3] : NAN);
      }
#pragma unroll
      for (int k = 0; k < AT; ++k)
        f(i0 + 128 * k, v[k]);
    }
  };

  /* ---- the greatest logit */
  float mx = -INFINITY;
  for_slice([&](unsigned, const float4 &v) { mx = fmaxf(fmaxf(mx, fmaxf(v.x, v.y)), fmaxf(v.z, v.w)); }); // a NaN never wins
#pragma unroll
  for (int o = 16; o; o >>= 1)
    mx = fmaxf(mx, __shfl_xor_sync(FULL, mx, o));
  if (lane == 0)
    sh.warp_max[warp] = mx;
  if (tid == 0)
    sh.count = sh.verdict = 0;
  __syncthreads();
  mx = sh.warp_max[0];
  for (int i = 1; i < SP_WARPS; ++i)
    mx = fmaxf(mx, sh.warp_max[i]);
  if (parts > 1) {
    cluster_wait();
    if (tid < parts)
      st_remote32(&sh.max_of[part], tid, __float_as_uint(mx));
    cluster_sync();
    for (int k = 0; k < parts; ++k)
      mx = fmaxf(mx, sh.max_of[k]);
  }
  auto tell = [&](unsigned id, double prob) {
    if (a.idx)
      a.idx[row] = id;
    if (a.idx_f)
      a.idx_f[row] = (float)id;
    if (a.prob)
      a.prob[row] = (float)prob;
  };
  if (mx == -INFINITY) { // nothing to draw from: the first token, as for the greatest of nothing
    if (part == 0 && tid == 0)
      tell(0, 0.0);
    return;
  }
  if (!(temperature > 0.0)) { // greedy
    temperature = 1.0;
    top_k = 1;
  }
  if (!(top_p > 0.0))
    top_k = 1;
  Weigher weight(mx, temperature);
  const bool has_k = top_k > 0 && top_k < a.n, has_p = top_p > 0.0 && top_p < 1.0;
  const bool whole = !has_k && !has_p && !(min_p > 0.0); // every token is kept
  if (tid == 0)
    sh.min_x = min_p > 0.0 ? weight.least_with(min_p) : -3.402823466e38f; // -inf is never kept

  /* ---- from which value up there are about SP_HEAD logits */
  const float per_bin = weight.c_hi * (SP_BINS / 46.f);
  auto bin_of = [&](float v) { return min(SP_BINS - 1, (int)fminf((mx - v) * per_bin, (float)SP_BINS)); };
  auto edge_of = [&](int bin) { return bin >= SP_BINS ? -3.402823466e38f : mx - (float)bin / per_bin; }; // the least value of the bins in front
  float head = -3.402823466e38f;
  if (a.n > SP_LIST) {
    sh.bins[tid] = 0;
    __syncthreads();
    const unsigned sub = part * SP_WARPS + warp;
    for (unsigned i0 = s0 + sub % SP_EVERY * 128; i0 < s1; i0 += 128 * SP_EVERY)
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const unsigned i = i0 + 32 * k + lane;
        const float v = i < s1 ? x[i] : NAN;
        if (v > -INFINITY)
          atomicAdd(&sh.bins[bin_of(v)], 1u);
      }
    __syncthreads();
    if (parts > 1)
      cluster_sync();
    uint32_t all = 0;
    for (int k = 0; k < parts; ++k)
      all += parts > 1 ? ld_remote32(&sh.bins[tid], k) : sh.bins[tid];
    sh.all_bins[tid] = all;
    __syncthreads();
    if (warp == 0) { // the last bin that the counts so far, times SP_EVERY, are not too many with
      unsigned run = 0, v[SP_BINS / 32];
#pragma unroll
      for (int k = 0; k < SP_BINS / 32; ++k)
        run += v[k] = sh.all_bins[lane * (SP_BINS / 32) + k];
      unsigned long long in_front = warp_scan(run, lane) - run;
      int last = 0; // bins in front of the edge
#pragma unroll
      for (int k = 0; k < SP_BINS / 32; ++k) {
        in_front += v[k];
        if (in_front * SP_EVERY <= SP_HEAD)
          last = lane * (SP_BINS / 32) + k + 1;
      }
      last = __reduce_max_sync(FULL, last);
      if (lane == 0)
        sh.from = edge_of(last);
    }
    __syncthreads();
    head = sh.from;
    weight.exact_from = fmaxf(weight.exact_from, head);
  } else {
    __syncthreads();
  }
  const float min_x = sh.min_x;

  /* Logits from `from` up to `below` into the list, which the first CTA gets; f(logit) for each of the others; what f adds up in each slice
   * goes to sh.sub of the first CTA. Returns how many are listed, ~0 if they are too many. */
  unsigned long long slice_sum = 0;
  unsigned n_above = 0;
  auto gather = [&](float from, float below, auto f) {
    if (tid == 0)
      sh.count = sh.n_above = 0;
    slice_sum = 0;
    n_above = 0;
    __syncthreads();
    for_slice([&](unsigned i, const float4 &v4) {
      const float v[4] = {v4.x, v4.y, v4.z, v4.w};
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const bool in = v[k] >= from && v[k] < below;
        if (!in)
          f(v[k]);
        const unsigned m = __ballot_sync(FULL, in);
        if (m) {
          unsigned at = 0;
          if (lane == 0)
            at = atomicAdd(&sh.count, (unsigned)__popc(m));
          at = __shfl_sync(FULL, at, 0) + __popc(m & ((1u << lane) - 1));
          if (in && at < SP_LIST) {
            sh.x[at] = v[k];
            sh.i[at] = i + k;
          }
        }
      }
    });
    slice_sum = warp_sum(slice_sum);
    n_above = __reduce_add_sync(FULL, n_above);
    if (lane == 0 && n_above)
      atomicAdd(&sh.n_above, n_above);
    __syncthreads();
    const unsigned own = sh.count;
    unsigned all = own;
    if (parts == 1) {
      if (lane == 0)
        sh.sub[warp] = slice_sum;
      if (tid == 0)
        sh.above[0] = sh.n_above;
      __syncthreads();
    } else {
      if (tid < parts) {
        st_remote32(&sh.counts[part], tid, own);
        st_remote32(&sh.above[part], tid, sh.n_above);
      }
      if (lane == 0)
        st_remote64(&sh.sub[part * SP_WARPS + warp], 0, slice_sum);
      cluster_sync();
      unsigned in_front = 0;
      all = 0;
      for (int k = 0; k < parts; ++k) {
        in_front += k < part ? sh.counts[k] : 0;
        all += sh.counts[k];
      }
      if (all <= SP_LIST && part > 0)
        for (unsigned i = tid; i < own; i += SP_THREADS) {
          st_remote32(&sh.x[in_front + i], 0, __float_as_uint(sh.x[i]));
          st_remote32(&sh.i[in_front + i], 0, sh.i[i]);
        }
      cluster_sync();
    }
    return all <= SP_LIST ? all : ~0u;
  };

  /* ---- the greatest logits listed, the others summed */
  const bool need_rest = whole || (has_p && !has_k);
  unsigned listed = gather(head, INFINITY, [&](float v) {
    if (v == INFINITY)
      ++n_above;
    else if (need_rest)
      slice_sum += weight(v);
  });
  const bool fits = listed != ~0u && mx < INFINITY; // an infinite logit is for the digits

  // Does the list do? Where that shows in the first CTA only, the others wait for its word.
  bool by_list = fits && (whole || has_p || has_k || min_x >= head);
  if (has_k && has_p && top_k > listed)
    by_list = false;
  const bool open = by_list && (has_k ? top_k > listed : has_p);
  const double u = a.u[row];
  auto goal_of = [&](unsigned long long total) { // the first sum above u * total
    const unsigned long long t = u > 0.0 ? (unsigned long long)fmin(u * (double)total, (double)total) + 1 : 1;
    return t < total ? t : total;
  };
  unsigned long long before, at;

  // The draw where it falls into a slice of the row: sh.sub holds the kept weights of the slices (in the first CTA).
  auto draw_in_slices = [&](auto kept) {
    const int n_sub = parts * SP_WARPS;
    if (warp == 0) {
      unsigned long long v[SP_MAX_PARTS * SP_WARPS / 32], run = 0;
#pragma unroll
      for (int k = 0; k < SP_MAX_PARTS * SP_WARPS / 32; ++k) {
        const int i = lane * (SP_MAX_PARTS * SP_WARPS / 32) + k;
        v[k] = i < n_sub ? sh.sub[i] : 0;
        run += v[k];
      }
      const unsigned long long upto = warp_scan(run, lane), total = __shfl_sync(FULL, upto, 31), goal = goal_of(total);
      const unsigned m = __ballot_sync(FULL, run > 0 && upto >= goal);
      if (lane == __ffs(m) - 1) {
        unsigned long long in_front = upto - run;
        int k = 0;
        while (k < SP_MAX_PARTS * SP_WARPS / 32 - 1 && !(v[k] && in_front + v[k] >= goal))
          in_front += v[k++];
        sh.digit = lane * (SP_MAX_PARTS * SP_WARPS / 32) + k;
        sh.before = in_front;
        sh.at = total;
      }
    }
    __syncthreads();
    const unsigned long long in_front = sh.before, total = sh.at, goal = goal_of(total);
    // the slice is dealt out to the warps again, in order
    const unsigned len = (a.sub_len / SP_WARPS + 31) / 32 * 32, q0 = sh.digit * a.sub_len, q1 = min(a.n, q0 + a.sub_len);
    const unsigned w0 = min(q1, q0 + warp * len), w1 = min(q1, w0 + len);
    unsigned long long mine = 0;
    for (unsigned i = w0 + lane; i < w1; i += 32)
      mine += kept(i, x[i]) ? weight(x[i]) : 0;
    mine = warp_sum(mine);
    if (lane == 0)
      sh.sum[warp] = mine;
    __syncthreads();
    unsigned long long run = in_front;
    for (int i = 0; i < warp; ++i)
      run += sh.sum[i];
    if (mine && run < goal && run + mine >= goal)
      for (unsigned i0 = w0; i0 < w1; i0 += 32) {
        const unsigned i = i0 + lane;
        const unsigned long long w = i < w1 && kept(i, x[i]) ? weight(x[i]) : 0, upto = run + warp_scan(w, lane);
        const unsigned m = __ballot_sync(FULL, w > 0 && upto >= goal);
        if (m) {
          if (lane == __ffs(m) - 1)
            tell(i, weight.exactly(x[i]) * SP_ONE / (double)total);
          break;
        }
        run = __shfl_sync(FULL, upto, 31);
      }
  };

  uint32_t cut = 1, cut_idx = 0xffffffffu; // tokens above `cut` are kept, of those at it the ones with an index up to cut_idx
  unsigned long long of_cut = 0;           // so many of those at the cut, the lowest indices; 0: no cut
  auto kept = [&](unsigned i, float v) {
    const uint32_t o = order_of(v);
    return o && (!of_cut || o > cut || (o == cut && i <= cut_idx)) && (v >= min_x || v == mx);
  };
  // over the list (in the first CTA)
  auto each = [&](bool count) {
    return [&, count](auto f) {
      for (unsigned i = tid; i < listed; i += SP_THREADS)
        f(order_of(sh.x[i]), count ? 1ull : weight(sh.x[i]));
    };
  };
  auto list_sum = [&](auto which) {
    unsigned long long sum = 0;
    for (unsigned i = tid; i < listed; i += SP_THREADS)
      sum += which(sh.i[i], sh.x[i]) ? weight(sh.x[i]) : 0;
    return cta_sum(sh, sum);
  };
  auto slices_sum = [&] {
    unsigned long long sum = 0;
    for (int i = 0; i < parts * SP_WARPS; ++i)
      sum += sh.sub[i];
    return sum;
  };
  auto cut_at = [&](uint32_t c, unsigned long long r) { // the first r tokens with value c
    if (c > cut || !of_cut || (c == cut && r < of_cut)) {
      cut = c;
      of_cut = r;
    }
  };
  auto cut_by_weight = [&](unsigned long long in_front, unsigned long long target) { // false: the list ends in front of the target
    const uint32_t c = descend(sh, 1, 32, true, target - in_front, each(false), &before, &at);
    if (in_front + before + at < target)
      return false;
    const unsigned long long w = weight(value_of(c));
    cut_at(c, (target - in_front - before + w - 1) / w);
    return true;
  };
  auto place_cut = [&] { // which of the equal ones are kept
    if (of_cut)
      cut_idx = descend(sh, 1, 20, false, of_cut, [&](auto f) {
        for (unsigned i = tid; i < listed; i += SP_THREADS)
          f(sh.i[i], order_of(sh.x[i]) == cut ? 1ull : 0ull);
      }, &before, &at);
  };
  auto list_to_slices = [&] {
    for (unsigned i = tid; i < listed; i += SP_THREADS)
      if (kept(sh.i[i], sh.x[i]))
        atomicAdd(&sh.sub[sh.i[i] / a.sub_len], weight(sh.x[i]));
    __syncthreads();
  };
  auto say = [&](unsigned word) { // the first CTA's word: 0 done, 1 one more pass from sh.from up to sh.upto, 2 by digits
    __syncthreads();
    if (parts > 1) {
      if (tid < parts) {
        st_remote32(&sh.from, tid, __float_as_uint(sh.from));
        st_remote32(&sh.upto, tid, __float_as_uint(sh.upto));
        st_remote32(&sh.verdict, tid, word);
      }
      cluster_sync();
    }
    return word;
  };
  unsigned word = by_list ? 0 : 2;
  unsigned long long target = 0;
  if (by_list && part == 0) {
    if (whole) {
      list_to_slices();
      draw_in_slices([](unsigned, float) { return true; });
      return;
    }
    bool enough = !has_k || top_k <= listed;
    if (has_k && top_k < listed) {
      cut = descend(sh, 1, 32, true, top_k, each(true), &before, &at);
      of_cut = top_k - before;
    }
    if (has_p && enough) {
      unsigned long long sum = list_sum([&](unsigned, float v) { return !of_cut || order_of(v) > cut; });
      sum += has_k ? of_cut * weight(value_of(cut)) : slices_sum();
      target = (unsigned long long)ceil(top_p * (double)sum);
      enough = cut_by_weight(0, target);
      if (!enough) { // about where it is: so much of the weight that is not listed lies in front of it
        const unsigned long long rest = slices_sum();
        if (warp == 0) {
          double v[SP_BINS / 32], run = 0.0;
#pragma unroll
          for (int k = 0; k < SP_BINS / 32; ++k) {
            const int b = lane * (SP_BINS / 32) + k;
            run += v[k] = edge_of(b) <= head ? sh.all_bins[b] * (double)exp2f(-(b + 0.5f) * (46.f / SP_BINS)) : 0.0;
          }
          double upto = run;
#pragma unroll
          for (int o = 1; o < 32; o *= 2) {
            const double t = __shfl_up_sync(FULL, upto, o);
            upto += lane >= o ? t : 0.0;
          }
          const double goal = __shfl_sync(FULL, upto, 31) * ((double)(target - (sum - rest)) / (double)rest);
          const unsigned m = __ballot_sync(FULL, run > 0.0 && upto >= goal);
          if (lane == (m ? __ffs(m) - 1 : 31)) {
            double in_front = upto - run;
            int k = 0;
            while (k < SP_BINS / 32 - 1 && in_front + v[k] < goal)
              in_front += v[k++];
            sh.digit = lane * (SP_BINS / 32) + k;
          }
        }
      }
    } else if (!enough && warp == 0) { // top_k of more tokens than are listed
      unsigned run = 0, v[SP_BINS / 32];
#pragma unroll
      for (int k = 0; k < SP_BINS / 32; ++k)
        run += v[k] = sh.all_bins[lane * (SP_BINS / 32) + k];
      const unsigned long long upto = warp_scan(run, lane);
      const unsigned m = __ballot_sync(FULL, run > 0 && upto * SP_EVERY >= top_k);
      if (lane == (m ? __ffs(m) - 1 : 31)) {
        unsigned long long in_front = upto - run;
        int k = 0;
        while (k < SP_BINS / 32 - 1 && (in_front + v[k]) * SP_EVERY < top_k)
          in_front += v[k++];
        sh.digit = lane * (SP_BINS / 32) + k;
      }
    }
    if (!enough && min_x >= head) // what passes min_p is listed, and in front of the cut
      enough = true;
    __syncthreads();
    if (!enough && tid == 0) { // the bins around that one
      const unsigned half = SP_AROUND / 2 / SP_EVERY;
      int hi = sh.digit, lo = hi + 1;
      for (unsigned c = 0; hi > 0 && edge_of(hi) < head && c + sh.all_bins[hi - 1] <= half;)
        c += sh.all_bins[--hi];
      for (unsigned c = 0; lo < SP_BINS && c + sh.all_bins[lo] <= half;)
        c += sh.all_bins[lo++];
      sh.upto = fminf(edge_of(hi), head);
      sh.from = edge_of(lo);
    }
    word = enough ? 0 : 1;
    if (open)
      word = say(word);
    if (word == 0) {
      place_cut();
      const unsigned long long total = list_sum(kept);
      const uint32_t id = descend(sh, 1, 20, false, goal_of(total), [&](auto f) {
        for (unsigned i = tid; i < listed; i += SP_THREADS)
          f(sh.i[i], kept(sh.i[i], sh.x[i]) ? weight(sh.x[i]) : 0);
      }, &before, &at);
      if (tid == 0)
        tell(id, weight.exactly(x[id]) * SP_ONE / (double)total);
    }
  } else if (open) {
    cluster_sync();
    word = sh.verdict;
  }
  if (word == 0)
    return;

  if (word == 1) {
    /* ---- one more pass: the logits around the cut listed, those above summed */
    __syncthreads();
    const float from = sh.from, below = sh.upto;
    listed = gather(from, below, [&](float v) {
      if (v >= below) {
        slice_sum += weight(v);
        ++n_above;
      }
    });
    word = listed == ~0u || min_x >= below ? 2 : 0;
    if (word == 0) {
      if (part == 0) {
        bool found;
        if (has_k) {
          unsigned above = 0;
          for (int k = 0; k < parts; ++k)
            above += sh.above[k];
          found = above < top_k && top_k <= above + listed;
          if (found) {
            const uint32_t c = descend(sh, 1, 32, true, top_k - above, each(true), &before, &at);
            cut_at(c, top_k - above - before);
          }
        } else {
          const unsigned long long above = slices_sum();
          found = above < target && cut_by_weight(above, target);
        }
        word = say(found ? 0 : 2);
        if (found) {
          place_cut();
          list_to_slices();
          draw_in_slices(kept);
        }
      } else {
        cluster_sync();
        word = sh.verdict;
      }
    }
    if (word == 0)
      return;
    cut = 1;
    of_cut = 0;
  }

  /* ---- the whole row by digits, every CTA its slices */
  auto each_of_row = [&](bool count) {
    return [&for_slice, &weight, count](auto f) {
      for_slice([&](unsigned, const float4 &v4) {
        const float v[4] = {v4.x, v4.y, v4.z, v4.w};
#pragma unroll
        for (int k = 0; k < 4; ++k)
          if (const uint32_t o = order_of(v[k]))
            f(o, count ? 1ull : weight(v[k]));
      });
    };
  };
  auto weigh = [&](auto which) { // over the cluster; each slice's sum into every CTA
    unsigned long long sum = 0;
    for_slice([&](unsigned i, const float4 &v4) {
      const float v[4] = {v4.x, v4.y, v4.z, v4.w};
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (which(i + k, v[k]))
          sum += weight(v[k]);
    });
    sum = warp_sum(sum);
    if (parts > 1) { // in every CTA
      if (lane < parts)
        st_remote64(&sh.sub[part * SP_WARPS + warp], lane, sum);
      cluster_sync();
    } else {
      if (lane == 0)
        sh.sub[warp] = sum;
      __syncthreads();
    }
    sum = 0;
    for (int i = 0; i < parts * SP_WARPS; ++i)
      sum += sh.sub[i];
    return sum;
  };
  if (parts > 1)
    cluster_sync(); // the first CTA is through with its histograms
  if (has_k) {
    cut = descend(sh, parts, 32, true, top_k, each_of_row(true), &before, &at);
    of_cut = top_k - before < at ? top_k - before : at; // all of them where there are fewer tokens than top_k
  }
  if (has_p) {
    const uint32_t above = cut;
    const bool all = !has_k;
    unsigned long long sum = weigh([&](unsigned, float v) { const uint32_t o = order_of(v); return all ? o != 0 : o > above; });
    if (has_k)
      sum += of_cut * weight(value_of(cut));
    if (parts > 1)
      cluster_sync(); // the sums are read before they are written again
    target = (unsigned long long)ceil(top_p * (double)sum);
    const uint32_t c = descend(sh, parts, 32, true, target, each_of_row(false), &before, &at);
    const unsigned long long w = weight(value_of(c)), r = target > before && w ? (target - before + w - 1) / w : 1;
    cut_at(c, r);
  }
  if (of_cut)
    cut_idx = descend(sh, parts, 20, false, of_cut, [&](auto f) {
      for_slice([&](unsigned i, const float4 &v4) {
        const float v[4] = {v4.x, v4.y, v4.z, v4.w};
#pragma unroll
        for (int k = 0; k < 4; ++k)
          if (order_of(v[k]) == cut)
            f(i + k, 1ull);
      });
    }, &before, &at);
  weigh(kept);
  if (part == 0)
    draw_in_slices(kept);
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
  if (!row_params && (!(temperature >= 0.0 && temperature <= 1e30) || !(top_p >= 0.0) || !(min_p >= 0.0 && min_p <= 1.0)))
    return set_error(NNTR_CUDA_ERR_INVALID, "sample: temperature %g, top_p %g, min_p %g; need temperature from 0 to 1e30, top_p >= 0, min_p from 0 to 1",
                     temperature, top_p, min_p);
  constexpr int smem = sizeof(SampleShared);
  static std::atomic<bool> set[64];
  int dev = 0;
  NNTR_CHECK_CUDA(cudaGetDevice(&dev));
  if (dev < 0 || dev >= 64 || !set[dev].load(std::memory_order_acquire)) {
    NNTR_CHECK_CUDA(cudaFuncSetAttribute(sample_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
    if (dev >= 0 && dev < 64)
      set[dev].store(true, std::memory_order_release);
  }
  int parts = 1;
  while (parts < SP_MAX_PARTS && rows * parts < 2 * sm_count() && n >= 4ll * SP_THREADS * parts)
    parts *= 2;
  const unsigned per_warp = (unsigned)((n + parts * SP_WARPS - 1) / (parts * SP_WARPS));
  SampleArgs a = {logits, u, row_params, ld, (unsigned)n, (per_warp + 127) / 128 * 128, 0, temperature, top_p, min_p, top_k, idx, idx_f, prob};
  a.vec = !(reinterpret_cast<uintptr_t>(logits) & 15) && (ld % 4 == 0 || rows == 1);
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[2];
  cfg.attrs = attr;
  if (flags & NNTR_CUDA_GEMV_PDL) {
    attr[cfg.numAttrs].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[cfg.numAttrs++].val.programmaticStreamSerializationAllowed = 1;
  }
  if (parts > 1) {
    attr[cfg.numAttrs].id = cudaLaunchAttributeClusterDimension;
    attr[cfg.numAttrs].val.clusterDim.x = parts;
    attr[cfg.numAttrs].val.clusterDim.y = attr[cfg.numAttrs].val.clusterDim.z = 1;
    ++cfg.numAttrs;
  }
  cfg.stream = st;
  cfg.gridDim = dim3((unsigned)(rows * parts));
  cfg.blockDim = dim3(SP_THREADS);
  cfg.dynamicSmemBytes = smem;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, sample_kernel, a);
  count_launch();
  return check_cuda(e, "sample launch");
}

} // namespace nntr
