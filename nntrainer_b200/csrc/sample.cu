// SPDX-License-Identifier: Apache-2.0
/**
 * @file  sample.cu
 * @brief A token per row of logits, drawn with temperature, top-k, top-p and min-p from a random number that the caller gives.
 *
 * With w_i = exp((x_i - max x) / T) and the tokens in descending order of x, the lowest index first among equals: the first top_k of
 * them are kept, of these the shortest prefix whose weights reach top_p times their sum, of these those with w_i >= min_p. The token is
 * the first kept one, in ascending order of the index, up to which the kept weights exceed u times their sum.
 *
 * A token is right or wrong, so the sums must not depend on their order: weights are whole multiples of 2^-44 (2^20 logits: 2^-43) in 64 bits. The ones that
 * count most (a few thousand of the greatest logits, down to 2^-14 of the greatest weight) are computed in double precision, the rest
 * of the row in fp32 to 2^-22 of themselves.
 *
 * A row is read for its greatest logit, an eighth of it for a histogram that says from which value up there are about SP_HEAD logits, and
 * again (from L2) for the list of these and the sum of the others. The first CTA of the row's cluster holds the list in shared memory and finds
 * the cuts and the draw by digits of eight bits, each a histogram. Where a cut lies below the list, the histogram says
 * about where; one more pass lists the logits around it and sums what is above, slice by slice. Where that does not do either (very many
 * equal logits, top_k and top_p both far down) the whole cluster goes by digits over the whole row.
 *
 * What bounds it: for a row the chain of passes (greatest logit, histogram, list, cuts, draw: five to eight barriers of the cluster or CTA
 * each), one row of 151936 logits with top_k 20 and top_p 0.95 14.0 us. Many rows: 128 of 201088 (103 MB) with top_p 0.9 and min_p 0.02 53 us, 1.9 TB/s, wait for
 * the loads of pass after pass (five of thirteen clocks between two instructions of a warp). No unit is the bound: issue slots 45 %, ALU
 * 25, FMA pipes 21. Half of the second reading comes from HBM once more, and 256 CTAs leave 40 of the 148 SMs with one in place of two (75000
 * clocks at work against 126000). As first built, all weights in double precision and digits over the whole row: 1240 and 2234 us.
 * Digits over the whole row as they are now, for 1 and 128 rows: top_k 20000 with top_p 0.9 161 and 964 us; temperature 1e-5 (below |greatest logit| / 7e5,
 * where weights are double precision throughout) 30 and 168, 24 at temperature 1; equal logits 29 and 132; top_p 0.9 of flat rows 170 and 747.
 */
#include "cluster.cuh"
#include "pipeline.cuh"

#include <algorithm>

namespace nntr {

namespace {

constexpr int SP_THREADS = 512, SP_WARPS = SP_THREADS / 32;
constexpr int SP_MAX_PARTS = 8;
static_assert(SP_THREADS == 512, "a thread per bin, two per digit");
constexpr int SP_LIST = 6144;              // logits that the list holds
constexpr int SP_HEAD = 2048;              // logits that it is meant for, the greatest ones
constexpr int SP_AROUND = 4400;            // ... and around a cut further down: three standard deviations of the estimate and more
constexpr int SP_FEW = 128;                // tokens that are compared each with each
constexpr int SP_BINS = 512;               // of the estimate, over 46 powers of two of the weight
constexpr int SP_EVERY = 8;                // every eighth block of 128 logits is in it
constexpr double SP_ONE = 17592186044416.0; // 2^44: fewer than 2^20 logits of the greatest weight stay in 64 bits
constexpr float SP_HIGH = 6.f, SP_LOW = 1.5f / 2097152.f; // the last bit of the one plus a weight is 2^-21, of the other plus up to 2^-22 either way 2^-44
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
  unsigned long long w[SP_LIST], few_w[SP_FEW];
  float x[SP_LIST];
  uint32_t i[SP_LIST], few_o[SP_FEW], few_i[SP_FEW];
  uint32_t hist[2][2][256]; // of a digit: the sum of its tokens' weights in two words; digit d at d % 8 * 32 + d / 8
  uint32_t bins[SP_BINS], all_bins[SP_BINS]; // of this CTA's part of the row, of the row
  unsigned long long sub[SP_MAX_PARTS * SP_WARPS], sum[SP_WARPS], before, at;
  float max_of[SP_MAX_PARTS], warp_max[SP_WARPS], min_x, from, upto;
  uint32_t counts[SP_MAX_PARTS], above[SP_MAX_PARTS], count, n_above, digit, verdict, few;
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
  float mx, exact_from, least; // the greatest logit; from here up in double precision; logits further down weigh as little as this one, nothing
  bool fp32;            // others in fp32; else all in double precision
  double top, per_t;
  unsigned n; // logits
  float c_hi, c_lo, m_hi, m_lo; // log2(e) / T, and times the greatest logit, each as a sum of two

  __device__ __forceinline__ Weigher(float mx_, double t, unsigned n_) : mx(mx_), top(mx_), per_t(1.0 / t), n(n_) {
    exact_from = fmaxf((float)(top - SP_EXACT_NATS * t), -3.402823466e38f);
    const double c = 1.4426950408889634 / t, m = c * top;
    c_hi = (float)c;
    c_lo = (float)(c - (double)c_hi);
    m_hi = (float)(rint(m * 8.0) * 0.125); // plus a small whole number it is exact
    m_lo = (float)(m - (double)m_hi);
    m_hi += n == SP_MAX_N ? 1.f : 0.f;
    fp32 = fabs(m) < 1048576.0 && c <= 3.402823466e38; // with a greatest logit of 0 m says nothing about c
    least = (float)(top - 60.0 / c);
    if (!fp32) { // it is not: few logits are that large against the temperature
      c_hi = c_lo = m_lo = least = 0.f; // what is in no order weighs 2^-60
      m_hi = 60.f;
      exact_from = -3.402823466e38f;
    }
  }
  /* the greatest weight: half of 2^44 where there are as many logits as can be, so that their sum is not 2^64 */
  __device__ __forceinline__ double one() const { return n == SP_MAX_N ? SP_ONE / 2 : SP_ONE; }
  __device__ __forceinline__ double exactly(float x) const { return x == mx ? 1.0 : x > -INFINITY ? exp(((double)x - top) * per_t) : 0.0; }
  __device__ __forceinline__ unsigned long long exact_one(float x) const { return __double2ull_rn(exactly(x) * one()); }
  /* Two logits, their weights rounded to whole multiples of 2^-44: of 2^-21 in the low bits of w + 6, what is left of that, of 2^-44 in those
   * of the rest + 1.5 * 2^-21. So most of it is fp32, two operations in one instruction, and sums of weights are sums of words. (64-bit shifts,
   * comparisons and selections run at half the rate: with them the reading of 128 rows took 1.6 times as long.) */
  __device__ __forceinline__ void in_fp32(float x0, float x1, uint32_t (&hi)[2], uint32_t (&lo)[2]) const {
    constexpr float MAGIC = 12582912.f; // 1.5 * 2^23: the sum's low bits are the nearest whole number
    x0 = fmaxf(x0, least), x1 = fmaxf(x1, least); // NaN is `least` too
    float y0 = -m_hi, y1 = -m_hi, g0 = -m_lo, g1 = -m_lo;
    fma2(y0, y1, x0, x1, c_hi, c_hi);
    fma2(g0, g1, x0, x1, c_lo, c_lo);
    const float2 t = add2(y0, y1, MAGIC, MAGIC), n = add2(t.x, t.y, -MAGIC, -MAGIC), s = add2(n.x, n.y, m_hi, m_hi);
    float f0 = -s.x, f1 = -s.y;
    fma2(f0, f1, x0, x1, c_hi, c_hi);
    const float2 f = add2(f0, f1, g0, g1);
    float q0 = 1.3398874413974103e-3f, q1 = q0, r0, r1;
    fma2(q0, q1, 1.535336190840639e-4f, 1.535336190840639e-4f, f.x, f.y);
    r0 = r1 = 9.618437357669995e-3f;
    fma2(r0, r1, q0, q1, f.x, f.y);
    q0 = q1 = 5.550332471126199e-2f;
    fma2(q0, q1, r0, r1, f.x, f.y);
    r0 = r1 = 2.4022647913628897e-1f;
    fma2(r0, r1, q0, q1, f.x, f.y);
    q0 = q1 = 6.931472028550653e-1f;
    fma2(q0, q1, r0, r1, f.x, f.y);
    r0 = r1 = 1.f;
    fma2(r0, r1, q0, q1, f.x, f.y);
    const float w0 = __uint_as_float(__float_as_uint(r0) + (__float_as_uint(t.x) << 23)), w1 = __uint_as_float(__float_as_uint(r1) + (__float_as_uint(t.y) << 23));
    const float2 a = add2(w0, w1, SP_HIGH, SP_HIGH), h = add2(a.x, a.y, -SP_HIGH, -SP_HIGH), l = add2(w0, w1, -h.x, -h.y), b = add2(l.x, l.y, SP_LOW, SP_LOW);
    hi[0] = __float_as_uint(a.x), hi[1] = __float_as_uint(a.y);
    lo[0] = __float_as_uint(b.x), lo[1] = __float_as_uint(b.y);
  }
  /* a sum of n weights from the sums of their words, for up to 128 of them */
  static __device__ __forceinline__ unsigned long long sum_of(uint32_t hi, uint32_t lo, int n) {
    return ((long long)(int)(hi - n * __float_as_uint(SP_HIGH)) << 23) + (int)(lo - n * __float_as_uint(SP_LOW));
  }
  __device__ __forceinline__ unsigned long long operator()(float x) const {
    if (x >= exact_from)
      return exact_one(x);
    uint32_t hi[2], lo[2];
    in_fp32(x, x, hi, lo);
    return sum_of(hi[0], lo[0], 1);
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
    h[tid >> 8][tid & 255] = 0;
    __syncthreads();
    each([&](const uint32_t(&key)[4], const unsigned long long(&w)[4]) { // four on their way at a time
      uint32_t old[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int d = key[k] >> shift & 255;
        old[k] = 0;
        if (w[k] && (unsigned long long)key[k] >> (shift + 8) == prefix)
          old[k] = atomicAdd(&h[0][d % 8 * 32 + d / 8], (uint32_t)w[k]);
      }
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int d = key[k] >> shift & 255;
        const uint32_t up = (uint32_t)(w[k] >> 32) + (old[k] + (uint32_t)w[k] < old[k]); // with the carry
        if (up && (unsigned long long)key[k] >> (shift + 8) == prefix)
          atomicAdd(&h[1][d % 8 * 32 + d / 8], up);
      }
    });
    if (parts > 1) {
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
      const int column = down ? 31 - lane : lane; // eight digits
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const int at8 = (down ? 7 - k : k) * 32 + column;
        v[k] = (unsigned long long)h[1][at8] << 32 | h[0][at8];
        run += v[k];
      }
      const unsigned long long upto = warp_scan(run, lane) + sum, all = __shfl_sync(FULL, upto, 31);
      const unsigned long long goal = target < all ? target : all;
      const unsigned m = __ballot_sync(FULL, run > 0 && upto >= goal);
      if (m == 0 ? lane == 0 : lane == __ffs(m) - 1) {
        unsigned long long in_front = upto - run, here = 0;
        int found = -1;
#pragma unroll
        for (int k = 0; k < 8; ++k)
          if (found < 0) {
            if (v[k] && in_front + v[k] >= goal) {
              found = k;
              here = v[k];
            } else {
              in_front += v[k];
            }
          }
        found = found < 0 ? 0 : found;
        sh.digit = column * 8 + (down ? 7 - found : found);
        sh.before = in_front;
        sh.at = here;
      }
    }
    __syncthreads();
    prefix = prefix << 8 | sh.digit;
    sum = sh.before;
    *at = sh.at;
  }
  *before = sum;
  return prefix;
}

} // namespace

__global__ void __launch_bounds__(SP_THREADS, 2) sample_kernel(SampleArgs a) {
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
  // this warp's slice of the row: the CTAs take slices in turn, so that none has all of the tokens that a model likes (low indices, often)
  const unsigned sub = warp * parts + part, s0 = min(a.n, sub * a.sub_len), s1 = min(a.n, s0 + a.sub_len);
  constexpr int AT = 4; // loads of a lane on their way at a time
  auto for_slice = [&](auto f, auto after) { // f(index, four logits); what is behind the slice is NaN; after() comes after AT of them
    for (unsigned i0 = s0 + 4 * lane; i0 - 4 * lane < s1; i0 += 128 * AT) {
      float v[AT][4];
#pragma unroll
      for (int k = 0; k < AT; ++k) {
        const unsigned i = i0 + 128 * k;
        if (a.vec && i + 4 <= s1) {
          const float4 w = *reinterpret_cast<const float4 *>(x + i);
          v[k][0] = w.x, v[k][1] = w.y, v[k][2] = w.z, v[k][3] = w.w;
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e)
            v[k][e] = i + e < s1 ? x[i + e] : NAN;
        }
      }
#pragma unroll
      for (int k = 0; k < AT; ++k)
        f(i0 + 128 * k, v[k]);
      after();
    }
  };
  auto nothing = [] {};

  /* ---- the greatest logit */
  float mx = -INFINITY;
  for_slice([&](unsigned, const float(&v)[4]) { mx = fmaxf(fmaxf(mx, fmaxf(v[0], v[1])), fmaxf(v[2], v[3])); }, nothing); // a NaN never wins
#pragma unroll
  for (int o = 16; o; o >>= 1)
    mx = fmaxf(mx, __shfl_xor_sync(FULL, mx, o));
  if (lane == 0)
    sh.warp_max[warp] = mx;
  __syncthreads();
  mx = sh.warp_max[lane % SP_WARPS];
#pragma unroll
  for (int o = SP_WARPS / 2; o; o >>= 1)
    mx = fmaxf(mx, __shfl_xor_sync(FULL, mx, o));
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
  Weigher weight(mx, temperature, a.n);
  const bool has_k = top_k > 0 && top_k < a.n, has_p = top_p > 0.0 && top_p < 1.0;
  const bool whole = !has_k && !has_p && !(min_p > 0.0); // every token is kept
  if (tid == SP_THREADS - 1)
    sh.min_x = min_p > 0.0 ? weight.least_with(min_p) : -3.402823466e38f; // -inf is never kept

  /* ---- from which value up there are about SP_HEAD logits */
  const float per_bin = (float)(1.4426950408889634 * SP_BINS / 46.0 * weight.per_t);
  auto bin_of = [&](float v) { return min(SP_BINS - 1, (int)fminf((mx - v) * per_bin, (float)SP_BINS)); };
  auto edge_of = [&](int bin) { return bin >= SP_BINS ? -3.402823466e38f : mx - (float)bin / per_bin; }; // the least value of the bins in front
  float head = -3.402823466e38f;
  const unsigned wanted = has_k ? min((unsigned)SP_HEAD, 2 * min(top_k, (unsigned)SP_HEAD) + 32) : SP_HEAD;
  if (a.n > SP_LIST) {
    sh.bins[tid] = 0;
    __syncthreads();
    for (unsigned i0 = s0 + sub % SP_EVERY * 128; i0 < s1; i0 += 128 * SP_EVERY * 4) {
      float v[4][4];
#pragma unroll
      for (int b = 0; b < 4; ++b)
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const unsigned i = i0 + 128 * SP_EVERY * b + 32 * k + lane;
          v[b][k] = i < s1 ? x[i] : NAN;
        }
#pragma unroll
      for (int b = 0; b < 4; ++b)
#pragma unroll
        for (int k = 0; k < 4; ++k)
          if (v[b][k] > -INFINITY)
            atomicAdd(&sh.bins[bin_of(v[b][k])], 1u);
    }
    __syncthreads();
    uint32_t all = sh.bins[tid];
    if (parts > 1) {
      cluster_sync();
      uint32_t of[SP_MAX_PARTS];
#pragma unroll
      for (int k = 0; k < SP_MAX_PARTS; ++k)
        of[k] = k < parts ? ld_remote32(&sh.bins[tid], k) : 0;
      all = 0;
#pragma unroll
      for (int k = 0; k < SP_MAX_PARTS; ++k)
        all += of[k];
    }
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
        if (in_front * SP_EVERY <= wanted)
          last = lane * (SP_BINS / 32) + k + 1;
      }
      last = __reduce_max_sync(FULL, last);
      if (lane == 0)
        sh.from = edge_of(last);
    }
    __syncthreads();
    head = sh.from;
  } else {
    __syncthreads();
  }
  const float min_x = sh.min_x;
  if (min_p > 0.0 && !(has_k && has_p)) // what is below fails min_p (top_k and top_p together refer to a sum that has it)
    head = fmaxf(head, min_x);
  if (weight.fp32)
    weight.exact_from = fmaxf(weight.exact_from, head);

  /* Logits that are `wanted` into the list of the first CTA; all, four at a time, to f(logits, for each whether it is in
   * the list); what f adds up in each slice goes to sh.sub of the first CTA. Returns how many are listed, ~0 if they are too many. Each CTA
   * has its own part of the list. */
  unsigned long long slice_sum = 0;
  unsigned n_above = 0;
  const unsigned room = SP_LIST / parts;
  auto gather = [&](auto wanted, auto f, auto after) {
    if (tid == 0)
      sh.count = sh.n_above = 0;
    slice_sum = 0;
    n_above = 0;
    __syncthreads();
    uint32_t to_x, to_i;
    asm("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(to_x) : "r"(smem_u32(&sh.x[part * room])));
    asm("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(to_i) : "r"(smem_u32(&sh.i[part * room])));
    for_slice([&](unsigned i, const float(&v)[4]) {
      bool in[4];
#pragma unroll
      for (int k = 0; k < 4; ++k)
        in[k] = wanted(v[k]);
      f(v, in);
      if (in[0] || in[1] || in[2] || in[3])
#pragma unroll
        for (int k = 0; k < 4; ++k)
          if (in[k]) {
            const unsigned at = atomicAdd(&sh.count, 1u);
            if (at < room) {
              asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(to_x + 4 * at), "f"(v[k]) : "memory");
              asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(to_i + 4 * at), "r"(i + k) : "memory");
            }
          }
    }, after);
    slice_sum = warp_sum(slice_sum);
    n_above = __reduce_add_sync(FULL, n_above);
    if (lane == 0 && n_above)
      atomicAdd(&sh.n_above, n_above);
    if (parts > 1) {
      if (lane == 0)
        st_remote64(&sh.sub[sub], 0, slice_sum);
      __syncthreads();
      if (tid < parts) {
        st_remote32(&sh.counts[part], tid, sh.count);
        st_remote32(&sh.above[part], tid, sh.n_above);
      }
      cluster_sync();
    } else {
      if (lane == 0)
        sh.sub[sub] = slice_sum;
      __syncthreads();
      if (tid == 0) {
        sh.counts[0] = sh.count;
        sh.above[0] = sh.n_above;
      }
      __syncthreads();
    }
    unsigned all = 0, most = 0, count[SP_MAX_PARTS];
#pragma unroll
    for (int k = 0; k < SP_MAX_PARTS; ++k) {
      count[k] = k < parts ? sh.counts[k] : 0;
      all += count[k];
      most = max(most, count[k]);
    }
    if (most > room)
      return ~0u;
    if (part == 0) { // the parts close up: an entry moves to a place that is not behind it, so that no later one is written over
      for (unsigned i0 = 0; i0 < (parts > 1 ? all : 0); i0 += SP_THREADS) {
        const unsigned i = i0 + tid;
        unsigned from_k = 0, in_front = 0;
#pragma unroll
        for (int k = 0; k < SP_MAX_PARTS; ++k)
          if (i >= in_front + count[k] && i < all) {
            in_front += count[k];
            from_k = k + 1;
          } else {
            break;
          }
        const unsigned at = from_k * room + i - in_front;
        const float xv = i < all ? sh.x[at] : 0.f;
        const uint32_t iv = i < all ? sh.i[at] : 0;
        __syncthreads();
        if (i < all) {
          sh.x[i] = xv;
          sh.i[i] = iv;
        }
      }
      __syncthreads();
      for (unsigned i = tid; i < all; i += SP_THREADS)
        sh.w[i] = weight(sh.x[i]);
      __syncthreads();
    }
    return all;
  };

  /* ---- the greatest logits listed, the others summed */
  const bool need_rest = whole || (has_p && !has_k);
  uint32_t sum_hi = 0, sum_lo = 0;
  auto add_rest = [&](const float(&v)[4], const bool(&in)[4]) { // what is not listed is below exact_from
    if (!need_rest)
      return;
#pragma unroll
    for (int k = 0; k < 4; k += 2) {
      uint32_t hi[2], lo[2];
      weight.in_fp32(in[k] ? -INFINITY : v[k], in[k + 1] ? -INFINITY : v[k + 1], hi, lo);
      sum_hi += hi[0] + hi[1];
      sum_lo += lo[0] + lo[1];
    }
  };
  unsigned listed = gather([&](float v) { return v >= head; }, add_rest, [&] {
    if (need_rest)
      slice_sum += Weigher::sum_of(sum_hi, sum_lo, 4 * AT);
    sum_hi = sum_lo = 0;
  });
  const bool fits = listed != ~0u && weight.fp32; // else: by digits
  const bool all_listed = head == -3.402823466e38f;

  // Does the list do? Where that shows in the first CTA only, the others wait for its word.
  bool by_list = fits && (whole || has_p || has_k || min_x >= head);
  const bool deep_k = has_k && top_k > listed && !all_listed; // the top_k-th is not in it
  if (deep_k && has_p)
    by_list = false;
  const bool open = by_list && (has_k ? deep_k : has_p);
  const double u = a.u[row];
  auto goal_of = [&](unsigned long long total) { // the first sum above u * total
    const unsigned long long t = u > 0.0 ? (unsigned long long)fmin(u * (double)total, (double)total) + 1 : 1;
    return t < total ? t : total;
  };
  unsigned long long before, at;

  uint32_t cut = 1, cut_idx = 0xffffffffu; // tokens above `cut` are kept, of those at it the ones with an index up to cut_idx
  unsigned long long of_cut = 0;           // so many of those at the cut, the lowest indices; 0: no cut
  auto kept = [&](unsigned i, float v) {
    const uint32_t o = order_of(v);
    return o && (!of_cut || o > cut || (o == cut && i <= cut_idx)) && (v >= min_x || v == mx);
  };

  // The draw where it falls into a slice of the row: sh.sub holds the kept weights of the slices (in the first CTA).
  auto draw_in_slices = [&] {
    const int n_sub = parts * SP_WARPS;
    constexpr int EACH = SP_MAX_PARTS * SP_WARPS / 32;
    if (warp == 0) {
      unsigned long long v[EACH], run = 0;
#pragma unroll
      for (int k = 0; k < EACH; ++k) {
        v[k] = lane * EACH + k < n_sub ? sh.sub[lane * EACH + k] : 0;
        run += v[k];
      }
      const unsigned long long upto = warp_scan(run, lane), total = __shfl_sync(FULL, upto, 31), goal = goal_of(total);
      const unsigned m = __ballot_sync(FULL, run > 0 && upto >= goal);
      if (lane == __ffs(m) - 1) {
        unsigned long long in_front = upto - run;
        int found = -1;
#pragma unroll
        for (int k = 0; k < EACH; ++k)
          if (found < 0) {
            if (v[k] && in_front + v[k] >= goal)
              found = k;
            else
              in_front += v[k];
          }
        sh.digit = lane * EACH + found;
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
            tell(i, weight.exactly(x[i]) * weight.one() / (double)total);
          break;
        }
        run = __shfl_sync(FULL, upto, 31);
      }
  };

  // over the list (in the first CTA)
  auto over_list = [&](auto key, auto w) { // for descend(): key(entry), w(entry)
    return [&sh, listed, tid, key, w](auto f) {
      for (unsigned i0 = tid; i0 < listed; i0 += 4 * SP_THREADS) {
        uint32_t k4[4];
        unsigned long long w4[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const unsigned i = i0 + k * SP_THREADS;
          k4[k] = i < listed ? key(i) : 0;
          w4[k] = i < listed ? w(i) : 0;
        }
        f(k4, w4);
      }
    };
  };
  // values by how far they lie below the greatest: fewer digits
  const uint32_t best = order_of(mx);
  auto depth = [&](unsigned i) { return best - order_of(sh.x[i]); };
  auto bits_down_to = [&](float v) { return max(1, 32 - __clz(best - max(1u, order_of(v)))); };
  const int index_bits = max(1, 32 - __clz(a.n - 1));
  auto weight_of = [&](unsigned i) { return sh.w[i]; };
  auto list_sum = [&](auto which) {
    unsigned long long sum = 0;
    for (unsigned i = tid; i < listed; i += SP_THREADS)
      sum += which(sh.i[i], sh.x[i]) ? sh.w[i] : 0;
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
  auto cut_by_count = [&](float least, unsigned k) {
    const uint32_t c = best - descend(sh, 1, bits_down_to(least), false, k, over_list(depth, [](unsigned) { return 1ull; }), &before, &at);
    cut_at(c, k - before);
  };
  auto cut_by_weight = [&](float least, unsigned long long in_front, unsigned long long target) { // false: the list ends in front of the target
    const uint32_t c = best - descend(sh, 1, bits_down_to(least), false, target - in_front, over_list(depth, weight_of), &before, &at);
    if (in_front + before + at < target)
      return false;
    const unsigned long long w = weight(value_of(c));
    cut_at(c, (target - in_front - before + w - 1) / w);
    return true;
  };
  auto place_cut = [&] { // which of the equal ones are kept
    if (of_cut)
      cut_idx = descend(sh, 1, index_bits, false, of_cut, over_list([&](unsigned i) { return sh.i[i]; }, [&](unsigned i) {
        return order_of(sh.x[i]) == cut ? 1ull : 0ull;
      }), &before, &at);
  };
  auto list_to_slices = [&] {
    for (unsigned i = tid; i < listed; i += SP_THREADS)
      if (kept(sh.i[i], sh.x[i]))
        atomicAdd(&sh.sub[sh.i[i] / a.sub_len], sh.w[i]);
    __syncthreads();
  };
  /* Where few tokens, no more than SP_FEW, lie above the cut and pass min_p (value `passes`): each is compared with each. all: the sum that
   * top_p refers to, if it is known; else it is that of the tokens top_k leaves, which all lie above the cut then. False: there are more. */
  auto among_few = [&](uint32_t passes, unsigned long long all, bool known) {
    const uint32_t least = has_p && !known ? cut : max(cut, passes); // that sum has the tokens too that min_p drops
    if (tid == 0)
      sh.few = 0;
    __syncthreads();
    for (unsigned i = tid; i < listed; i += SP_THREADS) {
      const uint32_t o = order_of(sh.x[i]);
      if (o >= least) {
        const unsigned at = atomicAdd(&sh.few, 1u);
        if (at < SP_FEW) {
          sh.few_o[at] = o;
          sh.few_i[at] = sh.i[i];
          sh.few_w[at] = sh.w[i];
        }
      }
    }
    __syncthreads();
    const int n = (int)sh.few;
    if (n > SP_FEW)
      return false;
    if (n <= 32) { // within a warp
      if (warp > 0)
        return true;
      const bool there = lane < n;
      const uint32_t o = there ? sh.few_o[lane] : 0, id = there ? sh.few_i[lane] : 0;
      const unsigned long long w = there ? sh.few_w[lane] : 0;
      unsigned rank = 0;
      unsigned long long in_front = 0;
      for (int j = 0; j < n; ++j) {
        const uint32_t oj = __shfl_sync(FULL, o, j), ij = __shfl_sync(FULL, id, j);
        const unsigned long long wj = __shfl_sync(FULL, w, j);
        const bool before = oj > o || (oj == o && ij < id);
        rank += before;
        in_front += before ? wj : 0;
      }
      bool mine = there && (!has_k || rank < top_k);
      if (has_p) {
        if (!known)
          all = warp_sum(mine ? w : 0);
        mine = mine && in_front < (unsigned long long)ceil(top_p * (double)all);
      }
      mine = mine && o >= passes;
      const unsigned long long held = mine ? w : 0;
      unsigned long long upto = 0;
      for (int j = 0; j < n; ++j) {
        const uint32_t ij = __shfl_sync(FULL, id, j);
        const unsigned long long wj = __shfl_sync(FULL, held, j);
        upto += ij <= id ? wj : 0;
      }
      const unsigned long long total = warp_sum(held), goal = goal_of(total);
      if (held && upto >= goal && upto - held < goal)
        tell(id, weight.exactly(value_of(o)) * weight.one() / (double)total);
      return true;
    }
    const bool there = tid < n;
    const uint32_t o = there ? sh.few_o[tid] : 0, id = there ? sh.few_i[tid] : 0;
    const unsigned long long w = there ? sh.few_w[tid] : 0;
    unsigned rank = 0;
    unsigned long long in_front = 0;
    if (warp * 32 < n)
#pragma unroll 4
      for (int j = 0; j < n; ++j) {
        const uint32_t oj = sh.few_o[j], ij = sh.few_i[j];
        const unsigned long long wj = sh.few_w[j];
        const bool before = oj > o || (oj == o && ij < id);
        rank += before;
        in_front += before ? wj : 0;
      }
    bool mine = there && (!has_k || rank < top_k);
    if (has_p) {
      if (!known)
        all = cta_sum(sh, mine ? w : 0);
      mine = mine && in_front < (unsigned long long)ceil(top_p * (double)all);
    }
    mine = mine && o >= passes;
    __syncthreads();
    if (there)
      sh.few_w[tid] = mine ? w : 0;
    const unsigned long long total = cta_sum(sh, mine ? w : 0), goal = goal_of(total);
    if (warp * 32 < n && __any_sync(FULL, mine)) {
      unsigned long long upto = 0;
#pragma unroll 4
      for (int j = 0; j < n; ++j) {
        const uint32_t ij = sh.few_i[j];
        const unsigned long long wj = sh.few_w[j];
        upto += ij <= id ? wj : 0;
      }
      if (mine && w && upto >= goal && upto - w < goal)
        tell(id, weight.exactly(value_of(o)) * weight.one() / (double)total);
    }
    return true;
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
      draw_in_slices();
      return;
    }
    const uint32_t least = min_x >= head ? order_of(min_x) : 1u; // what lies below fails min_p
    bool enough = !deep_k;
    unsigned long long sum = 0;
    if (has_p && !has_k) {
      sum = list_sum([](unsigned, float) { return true; }) + slices_sum();
      target = (unsigned long long)ceil(top_p * (double)sum);
    }
    const bool early = open && least > 1u && !deep_k; // whatever top_p says, the kept tokens are listed
    if (early)
      say(0);
    if (enough && (!has_p || has_k || least > 1u || all_listed) && among_few(least, sum, !has_k))
      return;
    if (has_k && top_k < listed) {
      cut_by_count(head, top_k);
      if (among_few(least, sum, !has_k))
        return;
    }
    if (has_p && enough) {
      if (has_k) {
        sum = list_sum([&](unsigned, float v) { return !of_cut || order_of(v) > cut; }) + of_cut * weight(value_of(cut));
        target = (unsigned long long)ceil(top_p * (double)sum);
      }
      enough = cut_by_weight(head, 0, target) || least > 1u; // what passes min_p is listed, and in front of any cut further down
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
            int found = SP_BINS / 32;
#pragma unroll
            for (int k = 0; k < SP_BINS / 32; ++k)
              if (found == SP_BINS / 32) {
                if (in_front + v[k] >= goal)
                  found = k;
                else
                  in_front += v[k];
              }
            sh.digit = min(SP_BINS - 1, lane * (SP_BINS / 32) + found);
          }
        }
      }
    } else if (!enough && warp == 0) { // top_k of more tokens than are listed
      unsigned run = 0;
      for (int k = 0; k < SP_BINS / 32; ++k)
        run += sh.all_bins[lane * (SP_BINS / 32) + k];
      const unsigned long long upto = warp_scan(run, lane);
      const unsigned m = __ballot_sync(FULL, run > 0 && upto * SP_EVERY >= top_k);
      if (lane == (m ? __ffs(m) - 1 : 31)) {
        unsigned long long in_front = upto - run;
        int k = 0;
        while (k < SP_BINS / 32 - 1 && (in_front + sh.all_bins[lane * (SP_BINS / 32) + k]) * SP_EVERY < top_k)
          in_front += sh.all_bins[lane * (SP_BINS / 32) + k++];
        sh.digit = lane * (SP_BINS / 32) + k;
      }
    }
    enough = enough || least > 1u;
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
    if (open && !early)
      say(word);
    if (word == 0) {
      if (of_cut && among_few(least, sum, true))
        return;
      place_cut();
      const unsigned long long total = list_sum(kept);
      const uint32_t id = descend(sh, 1, index_bits, false, goal_of(total), over_list([&](unsigned i) { return sh.i[i]; }, [&](unsigned i) {
        return kept(sh.i[i], sh.x[i]) ? sh.w[i] : 0;
      }), &before, &at);
      if (tid == 0)
        tell(id, weight.exactly(x[id]) * weight.one() / (double)total);
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
    listed = gather([&](float v) { return v >= from && v < below; }, [&](const float(&v)[4], const bool(&)[4]) {
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (v[k] >= below) {
          slice_sum += weight(v[k]);
          ++n_above;
        }
    }, nothing);
    word = listed == ~0u || min_x >= below ? 2 : 0;
    if (word == 0) {
      if (part == 0) {
        bool found;
        if (has_k) {
          unsigned above = 0;
          for (int k = 0; k < parts; ++k)
            above += sh.above[k];
          found = above < top_k && top_k <= above + listed;
          if (found)
            cut_by_count(from, top_k - above);
        } else {
          const unsigned long long above = slices_sum();
          found = above < target && cut_by_weight(from, above, target);
        }
        word = say(found ? 0 : 2);
        if (found) {
          place_cut();
          list_to_slices();
          draw_in_slices();
        }
      } else {
        cluster_sync();
        word = sh.verdict;
      }
    }
    if (word == 0)
      return;
    cut = 1;
    cut_idx = 0xffffffffu;
    of_cut = 0;
  }

  /* ---- the whole row by digits, every CTA its slices */
  auto over_row = [&](auto key, auto w) { // key(index, logit), w(logit)
    return [&, key, w](auto f) {
      for_slice([&](unsigned i, const float(&v)[4]) {
        uint32_t k4[4];
        unsigned long long w4[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          k4[k] = key(i + k, v[k]);
          w4[k] = order_of(v[k]) ? w(v[k]) : 0;
        }
        f(k4, w4);
      }, nothing);
    };
  };
  auto by_value = [](unsigned, float v) { return order_of(v); };
  auto weigh = [&](auto which) { // over the cluster; each slice's sum into every CTA
    unsigned long long sum = 0;
    for_slice([&](unsigned i, const float(&v)[4]) {
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (which(i + k, v[k]))
          sum += weight(v[k]);
    }, nothing);
    sum = warp_sum(sum);
    if (parts > 1) { // in every CTA
      if (lane < parts)
        st_remote64(&sh.sub[sub], lane, sum);
      cluster_sync();
    } else {
      if (lane == 0)
        sh.sub[sub] = sum;
      __syncthreads();
    }
    return slices_sum();
  };
  __syncthreads();
  if (parts > 1)
    cluster_sync(); // the first CTA is through with its histograms
  if (has_k) {
    cut = descend(sh, parts, 32, true, top_k, over_row(by_value, [](float) { return 1ull; }), &before, &at);
    of_cut = top_k - before < at ? top_k - before : at; // all of them where there are fewer tokens than top_k
  }
  if (has_p) {
    const uint32_t above = has_k ? cut : 0;
    unsigned long long sum = weigh([&](unsigned, float v) { return order_of(v) > above; });
    if (has_k)
      sum += of_cut * weight(value_of(cut));
    if (parts > 1)
      cluster_sync(); // the sums are read before they are written again
    target = (unsigned long long)ceil(top_p * (double)sum);
    const uint32_t c = descend(sh, parts, 32, true, target, over_row(by_value, [&](float v) { return weight(v); }), &before, &at);
    const unsigned long long w = weight(value_of(c)), r = target > before && w ? (target - before + w - 1) / w : 1;
    cut_at(c, r);
  }
  if (of_cut)
    cut_idx = descend(sh, parts, index_bits, false, of_cut, over_row([](unsigned i, float) { return i; }, [&](float v) {
      return order_of(v) == cut ? 1ull : 0ull;
    }), &before, &at);
  __syncthreads();
  weigh(kept);
  if (part == 0)
    draw_in_slices();
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
  static SmemOptIn opt_in;
  if (const int rc = opt_in(sample_kernel, smem))
    return rc;
  int parts = 1;
  while (parts < SP_MAX_PARTS && rows * parts <= sm_count() && n >= 4ll * SP_THREADS * parts)
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
