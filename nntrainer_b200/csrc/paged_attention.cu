// SPDX-License-Identifier: Apache-2.0
/**
 * @file  paged_attention.cu
 * @brief Attention of the new tokens of a batch of sequences over a key/value cache in pages: few tokens of a sequence (one, or a
 *        draft's) here; launch_paged_attention() is the entry for all.
 *
 *   s_j = q . k_j / sqrt(head_dim) for the rows j the query at position p sees: j <= p and (j > p - window or j < first_tokens)
 *   out = sum_j exp(s_j - m) v_j / (sum_j exp(s_j - m) + exp(sink - m)), m = max_j s_j; zeros where nothing is seen
 *
 * Scores, maxima, sums and results are fp32. The probabilities are rounded to the cache's 16-bit type, the operand type of the
 * tensor cores (2^-11 or 2^-8 of each, which the sum over the rows averages out); what they may be: Weights in paged_attention.cuh.
 */
#include "cluster.cuh"
#include "paged_attention.cuh"
#include "pipeline.cuh"
#include "tma_map.cuh"

#include <algorithm>
#include <climits>

namespace nntr {

__device__ int g_paged_attn_status = 0;

int read_paged_attn_status(int *out, bool clear) {
  int v = 0;
  NNTR_CHECK_CUDA(cudaMemcpyFromSymbol(&v, g_paged_attn_status, sizeof(int)));
  if (v && clear) {
    const int zero = 0;
    NNTR_CHECK_CUDA(cudaMemcpyToSymbol(g_paged_attn_status, &zero, sizeof(int)));
  }
  *out = v;
  return NNTR_CUDA_OK;
}

/* ------------------------------------------------------ a few query rows */

/* Rows of a tile are (token, query head of the kv head's group), 16 of them: one M of the warp MMA. Every warp takes blocks of 16
 * cache rows in turn through a ring of its own, which one lane fills by TMA (a box of 16 rows and 64 dimensions), so that nothing but the
 * end is shared: scores of the block, probabilities straight from the accumulators to the operand of the second product. The
 * warps of a CTA join through shared memory, the CTAs of a cluster, which share the cache rows of one (sequence, kv head, tile),
 * through each other's.
 * Bandwidth bounds it: 2 * 2 * head_dim bytes per cache row and kv head. 64 streams of 150 to 8192 rows, 8 kv heads of 128: 172 us, 6444
 * GB/s, 0.99 of a copy's rate; 64 of 8192 rows 304 us, 7071 GB/s. One of 500 rows: 6.2 us, launch, first loads and join. Drafts, 16 x 5 tokens
 * of 32 heads on 8 at 2000 rows: 32 us where the bytes take 20 (two tiles read the same rows, the second time from L2); 16 x 9 by the other kernel 36. */
constexpr int PD_KEYS = 16; // of a block: no more than the smallest page
constexpr uint32_t PD_POLLS = 1u << 22;
template <int HD, int W> struct PdCfg { // W warps
  static constexpr int STAGES = HD == 128 ? 3 : 6;
  static constexpr int KV_BYTES = PD_KEYS * HD * 2; // [64 dimensions of HD][row][128 B], 128-byte swizzle
  static constexpr int RING = STAGES * 2 * KV_BYTES; // of a warp
  static_assert(RING >= (16 * HD + 32) * 4 && RING % 1024 == 0, "the warps' parts, O and (m, l), lie in the rings' place");
  // parts of the elements that a CTA joins (four columns of a row), from each of up to 16 CTAs: O, then (m, l) of each
  static constexpr int PARTS = 16 * HD / 4 + 16, PART_ML = PARTS * 16, OFF_PART = W * RING, OFF_BARS = OFF_PART + PARTS * 24;
  static constexpr int SMEM = OFF_BARS + W * STAGES * 8 + 16;
};

template <typename T> __device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1);
template <> __device__ __forceinline__ void mma16816<__half>(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <> __device__ __forceinline__ void mma16816<__nv_bfloat16>(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldsm4t(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}

__device__ __forceinline__ float max_nan(float a, float b) { // NaN if one of them is
  float d;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
  return d;
}

/* Parts of a row's result, four of O's columns, joined one after the other, up to four on their way at a time: load(i, &v, &ml). */
struct Joined {
  float4 sum;
  float m, l;

  template <class Load> __device__ __forceinline__ Joined(int n, Load load) : sum(make_float4(0.f, 0.f, 0.f, 0.f)), m(-INFINITY), l(0.f) {
    for (int i0 = 0; i0 < n; i0 += 4) {
      float4 v[4];
      float2 ml[4];
#pragma unroll
      for (int k = 0; k < 4; ++k)
        load(min(i0 + k, n - 1), &v[k], &ml[k]);
      float big = m;
#pragma unroll
      for (int k = 0; k < 4; ++k)
        big = fmaxf(big, ml[k].x);
      if (big == -INFINITY)
        continue;
      const float keep = ex2(m - big);
      sum = make_float4(sum.x * keep, sum.y * keep, sum.z * keep, sum.w * keep);
      l *= keep;
      m = big;
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (i0 + k < n) {
          const float w = ex2(ml[k].x - big);
          sum = make_float4(sum.x + w * v[k].x, sum.y + w * v[k].y, sum.z + w * v[k].z, sum.w + w * v[k].w);
          l += w * ml[k].y;
        }
    }
  }
};

template <typename T, int HD, int W>
__global__ void __launch_bounds__(W * 32)
paged_attention_few_kernel(const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap, AttendArgs a, PagedGeom g,
                           PagedBatch s) {
  using Cfg = PdCfg<HD, W>;
  extern __shared__ __align__(1024) uint8_t smem[];
  const int lane = threadIdx.x & 31, warp = __shfl_sync(FULL, threadIdx.x >> 5, 0);
  const int parts = cluster_size(), part = cluster_rank();
  const int tile = blockIdx.x / parts, h = blockIdx.y;
  const uint32_t bars = smem_u32(smem) + Cfg::OFF_BARS + warp * Cfg::STAGES * 8;
  volatile int *abort_flag = reinterpret_cast<volatile int *>(smem + Cfg::OFF_BARS + W * Cfg::STAGES * 8);
  pdl_launch_dependents();
  if (lane == 0) {
    for (int i = 0; i < Cfg::STAGES; ++i)
      mbar_init(bars + 8 * i, 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (threadIdx.x == 0)
    *abort_flag = 0;
  if (threadIdx.x == 0) {
    asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&kmap)));
    asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&vmap)));
  }
  if (parts > 1)
    cluster_arrive(); // every CTA has started before one writes into another
  pdl_wait();
  // Long contexts begin first: of up to 128 sequences (one per thread) the one with as many longer ones as CTAs are in front
  int seq = blockIdx.z;
  SeqRows r;
  if (s.batch > 1 && s.batch <= 128) {
    int *rows_of = reinterpret_cast<int *>(smem);
    int4 *chosen = reinterpret_cast<int4 *>(rows_of + 128);
    const int b = threadIdx.x;
    int4 mine = make_int4(b, 0, 0, INT_MIN);
    if (b < s.batch)
      mine = make_int4(b, __ldg(s.row_start + b), __ldg(s.row_start + b + 1), __ldg(s.context + b));
    if (b < 128)
      rows_of[b] = mine.w;
    __syncthreads();
    int longer = 0;
#pragma unroll 4
    for (int i = 0; i < s.batch; i += 4) {
      const int4 v = *reinterpret_cast<const int4 *>(rows_of + i);
      longer += (v.x > mine.w || (v.x == mine.w && i < b)) + (v.y > mine.w || (v.y == mine.w && i + 1 < b)) +
                (v.z > mine.w || (v.z == mine.w && i + 2 < b)) + (v.w > mine.w || (v.w == mine.w && i + 3 < b));
    }
    if (b < s.batch && longer == (int)blockIdx.z)
      *chosen = mine;
    __syncthreads();
    const int4 it = *chosen;
    seq = __shfl_sync(FULL, it.x, 0);
    r = seq_rows(s, it.y, it.z, it.w);
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); // the rings begin here
  } else {
    r = seq_rows(s, seq);
  }
  __syncthreads();
  if (r.bad && threadIdx.x == 0)
    atomicExch(&g_paged_attn_status, NNTR_CUDA_ERR_INVALID);
  const int G = g.hq / g.hkv, rows = min(16, r.n * G - tile * 16);
  if (rows <= 0) { // every CTA of the cluster alike
    if (parts > 1)
      cluster_wait();
    return;
  }
  const int tok0 = tile * 16 / G, tok1 = (tile * 16 + rows - 1) / G;
  const Sight sight(r.pos + tok0, r.pos + tok1, a.window, a.first, PD_KEYS);

  const uint32_t ring = smem_u32(smem) + warp * Cfg::RING;
  const int n_mine = sight.blocks > part * W + warp ? (sight.blocks - part * W - warp + parts * W - 1) / (parts * W) : 0;
  auto my_block = [&](int i) { return sight.block((i * parts + part) * W + warp); };
  // a lane keeps the page of one of the next 32 blocks, so that the way over the page table is taken once for all of them
  int page = 0;
  auto fetch = [&](int i) {
    if (i >= n_mine)
      return;
    if (i % 32 == 0 && i + lane < n_mine) {
      page = __ldg(s.table + (size_t)seq * s.ld_table + (my_block(i + lane) * PD_KEYS >> g.page_shift));
      if ((unsigned)page >= (unsigned)g.n_pages) {
        atomicExch(&g_paged_attn_status, NNTR_CUDA_ERR_INVALID);
        page = g.n_pages; // outside the map: zeros
      }
    }
    const int from = __shfl_sync(FULL, page, i % 32), row = my_block(i) * PD_KEYS & ((1 << g.page_shift) - 1);
    if (elected()) {
      const uint32_t bar = bars + 8 * (i % Cfg::STAGES), dst = ring + (i % Cfg::STAGES) * 2 * Cfg::KV_BYTES;
      mbar_expect_tx(bar, 2 * Cfg::KV_BYTES);
#pragma unroll
      for (int c = 0; c < HD / 64; ++c) {
        tma_box4(dst + c * 2048, &kmap, 64 * c, row, h, from, bar);
        tma_box4(dst + Cfg::KV_BYTES + c * 2048, &vmap, 64 * c, row, h, from, bar);
      }
    }
  };
  for (int i = 0; i < Cfg::STAGES - 1; ++i)
    fetch(i);

  // this lane's two rows: lane / 4 and 8 more
  const int gr = lane >> 2, gc = lane & 3;
  int row_pos[2];
  uint32_t qf[HD / 16][4];
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const int row = gr + 8 * k, flat = tile * 16 + row, tok = flat / G;
    row_pos[k] = row < rows ? r.pos + tok : -1;
    const T *qr = static_cast<const T *>(a.q) + (r.first + min(tok, tok1)) * a.ld_q + (size_t)(h * G + flat % G) * g.hd;
#pragma unroll
    for (int c = 0; c < HD / 16; ++c)
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const int col = 16 * c + 8 * u + 2 * gc;
        qf[c][k + 2 * u] = row < rows && col < g.hd ? *reinterpret_cast<const uint32_t *>(qr + col) : 0u;
      }
  }

  float o[HD / 8][4], m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
#pragma unroll
  for (int c = 0; c < HD / 8; ++c)
    o[c][0] = o[c][1] = o[c][2] = o[c][3] = 0.f;
  for (int i = 0; i < n_mine; ++i) {
    fetch(i + Cfg::STAGES - 1);
    if (!mbar_wait_warp(bars + 8 * (i % Cfg::STAGES), i / Cfg::STAGES & 1, abort_flag, &g_paged_attn_status, PD_POLLS, 2048))
      break;
    const uint32_t kt = ring + (i % Cfg::STAGES) * 2 * Cfg::KV_BYTES, vt = kt + Cfg::KV_BYTES;
    const int j0 = my_block(i) * PD_KEYS;
    if (!(j0 + PD_KEYS - 1 <= sight.hi && (j0 >= sight.from || j0 + PD_KEYS <= sight.first))) {
      // rows that nobody sees meet probabilities of zero: what they hold must be finite
      for (int k = lane; k < Cfg::KV_BYTES / 16; k += 32)
        if (!sight.row_read(j0 + (k >> 3 & (PD_KEYS - 1))))
          sts128(vt + 16 * k, 0, 0, 0, 0);
      __syncwarp();
    }
    float sc[2][4] = {}, odd[2][4] = {}; // two sums each: shorter chains
    { // four 8 x 8 matrices: keys 0-7 and 8-15, each with the lower and the upper 8 of 16 dimensions
      const int row = (lane & 7) + ((lane >> 4) << 3);
#pragma unroll
      for (int c = 0; c < HD / 16; ++c) {
        uint32_t b[4];
        ldsm4(b, kt + (c >> 2) * 2048 + row * 128 + (((2 * (c & 3) + ((lane >> 3) & 1)) ^ (row & 7)) << 4));
        mma16816<T>(c & 1 ? odd[0] : sc[0], qf[c], b[0], b[1]);
        mma16816<T>(c & 1 ? odd[1] : sc[1], qf[c], b[2], b[3]);
      }
    }
    const bool whole = j0 + PD_KEYS - 1 <= sight.lo && (j0 > sight.hi - sight.window || j0 + PD_KEYS <= a.first);
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int e = 0; e < 4; ++e)
        sc[t][e] += odd[t][e];
    if (!whole)
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int j = j0 + 8 * t + 2 * gc + (e & 1), p = row_pos[e >> 1];
          sc[t][e] = j <= p && (j > p - a.window || j < a.first) ? sc[t][e] : -INFINITY;
        }
    uint32_t pf[4];
    float sum[2];
    // A row's probabilities refer to a maximum m that is taken in the first block that it sees something of, and where rows are masked. Other
    // blocks go by the m there is; what they give shows whether it does. If not they begin again, with the maximum.
    for (bool afresh = !whole || __any_sync(FULL, m[0] == -INFINITY || m[1] == -INFINITY);; afresh = true) {
      if (afresh) {
        float mx[2], keep[2];
#pragma unroll
        for (int k = 0; k < 2; ++k)
          mx[k] = max_nan(max_nan(sc[0][2 * k], sc[0][2 * k + 1]), max_nan(sc[1][2 * k], sc[1][2 * k + 1]));
#pragma unroll
        for (int d = 1; d < 4; d *= 2)
#pragma unroll
          for (int k = 0; k < 2; ++k)
            mx[k] = max_nan(mx[k], __shfl_xor_sync(FULL, mx[k], d));
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          float big = max_nan(m[k], mx[k] * a.scale_log2);
          if (!(big < INFINITY)) { // a score that is no number or infinite, maybe the only one: the row's result is NaN
            big = INFINITY;
            l[k] = NAN;
          }
          keep[k] = big > m[k] ? ex2(m[k] - big) : 1.f;
          m[k] = big;
          l[k] *= keep[k];
        }
        if (__any_sync(FULL, keep[0] != 1.f || keep[1] != 1.f))
#pragma unroll
          for (int c = 0; c < HD / 8; ++c) {
            o[c][0] *= keep[0];
            o[c][1] *= keep[0];
            o[c][2] *= keep[1];
            o[c][3] *= keep[1];
          }
      }
#pragma unroll
      for (int k = 0; k < 2; ++k) { // the lane's two rows
        const float base = m[k] == -INFINITY ? 0.f : m[k] - Weights<T>::LIFT; // nothing seen yet: all weights are 2^(-inf)
        const float p0 = ex2(fmaf(sc[0][2 * k], a.scale_log2, -base)), p1 = ex2(fmaf(sc[0][2 * k + 1], a.scale_log2, -base)),
                    p2 = ex2(fmaf(sc[1][2 * k], a.scale_log2, -base)), p3 = ex2(fmaf(sc[1][2 * k + 1], a.scale_log2, -base));
        sum[k] = (p0 + p1) + (p2 + p3);
        pf[k] = pack2<T>(p0, p1);
        pf[k + 2] = pack2<T>(p2, p3);
      }
      if (afresh || !__any_sync(FULL, sum[0] > Weights<T>::MOST || sum[1] > Weights<T>::MOST))
        break;
    }
    l[0] += sum[0];
    l[1] += sum[1];
    { // keys 0-7 and 8-15 of eight dimensions, then of the next eight
      const int row = lane & 15;
#pragma unroll
      for (int c = 0; c < HD / 16; ++c) {
        uint32_t b[4];
        ldsm4t(b, vt + (c >> 2) * 2048 + row * 128 + (((2 * (c & 3) + (lane >> 4)) ^ (row & 7)) << 4));
        mma16816<T>(o[2 * c], pf, b[0], b[1]);
        mma16816<T>(o[2 * c + 1], pf, b[2], b[3]);
      }
    }
    loads_before_refill(); // the slot is read: the copies of the next round may fill it
    __syncwarp();
  }
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    l[k] += __shfl_xor_sync(FULL, l[k], 1);
    l[k] += __shfl_xor_sync(FULL, l[k], 2);
  }
  if (*abort_flag) // copies in flight get time to land before the rings are used otherwise
    for (int i = 0; i < 1000; ++i)
      __nanosleep(1000);

  /* ---- the warps' parts, then the CTAs': each a row's O, m and l; the rings are free */
  __syncthreads();
  float *mine = reinterpret_cast<float *>(smem + warp * Cfg::RING);
#pragma unroll
  for (int c = 0; c < HD / 8; ++c)
#pragma unroll
    for (int k = 0; k < 2; ++k)
      *reinterpret_cast<float2 *>(mine + (gr + 8 * k) * HD + 8 * c + 2 * gc) = make_float2(o[c][2 * k], o[c][2 * k + 1]);
  if (gc == 0)
#pragma unroll
    for (int k = 0; k < 2; ++k)
      *reinterpret_cast<float2 *>(mine + 16 * HD + 2 * (gr + 8 * k)) = make_float2(m[k], l[k]);
  __syncthreads();
  float *cta = reinterpret_cast<float *>(smem + Cfg::OFF_PART);
  const uint32_t cta_addr = smem_u32(cta);
  auto store = [&](int row, int col, const Joined &j) {
    const int flat = tile * 16 + row, head = h * G + flat % G;
    float total = j.l;
    if (a.sink && j.m > -INFINITY)
      total += ex2(a.sink[head] * LOG2E - (j.m - Weights<T>::LIFT));
    const float inv = total == 0.f ? 0.f : 1.f / total;
    const float4 f = make_float4(j.sum.x * inv, j.sum.y * inv, j.sum.z * inv, j.sum.w * inv);
    const long long e = (r.first + flat / G) * a.ld_out + (long long)head * g.hd + col;
    if (a.out_f32)
      *reinterpret_cast<float4 *>(static_cast<float *>(a.out) + e) = f;
    else
      *reinterpret_cast<uint2 *>(static_cast<T *>(a.out) + e) = make_uint2(pack2<T>(f.x, f.y), pack2<T>(f.z, f.w));
  };
  if (parts > 1) {
    cluster_wait(); // for the start
    if (*abort_flag)
      raise_in_cluster(smem_u32(const_cast<int *>(abort_flag)));
  }
  const bool gave_up = parts == 1 && *abort_flag; // then the result stays as it is
  // element i of the result (four columns of a row) is joined by CTA i / share of the cluster, which gets every CTA's part of it
  const int elements = rows * (HD / 4), share = (elements + parts - 1) / parts;
  for (int i = threadIdx.x; i < elements; i += W * 32) {
    const int row = i / (HD / 4), col = 4 * (i % (HD / 4));
    const Joined j(W, [&](int k, float4 *v, float2 *ml) {
      const float *p = reinterpret_cast<const float *>(smem + k * Cfg::RING);
      *v = *reinterpret_cast<const float4 *>(p + row * HD + col);
      *ml = *reinterpret_cast<const float2 *>(p + 16 * HD + 2 * row);
    });
    if (parts > 1) {
      const int owner = i / share, at = part * share + i % share;
      st_cluster4(cta_addr + 16u * at, owner, j.sum);
      uint32_t remote;
      asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(cta_addr + Cfg::PART_ML + 8u * at), "r"(owner));
      asm volatile("st.shared::cluster.v2.f32 [%0], {%1,%2};" ::"r"(remote), "f"(j.m), "f"(j.l) : "memory");
    } else if (col < g.hd && !gave_up) {
      store(row, col, j);
    }
  }
  if (parts == 1)
    return;
  cluster_sync(); // behind it nobody touches another's memory
  if (!*abort_flag)
    for (int k = threadIdx.x; k < share && part * share + k < elements; k += W * 32) {
      const int i = part * share + k, row = i / (HD / 4), col = 4 * (i % (HD / 4));
      if (col < g.hd)
        store(row, col, Joined(parts, [&](int q, float4 *v, float2 *ml) {
                *v = *reinterpret_cast<const float4 *>(cta + 4 * (q * share + k));
                *ml = *reinterpret_cast<const float2 *>(reinterpret_cast<const uint8_t *>(cta) + Cfg::PART_ML + 8 * (q * share + k));
              }));
    }
}

/* ------------------------------------------------------------------ launch */

template <typename T, int HD, int W>
static int launch_few(const AttendArgs &a, const PagedGeom &g, const PagedBatch &s, unsigned max_rows, int tiles, unsigned flags, cudaStream_t st) {
  auto kernel = paged_attention_few_kernel<T, HD, W>;
  constexpr int smem = PdCfg<HD, W>::SMEM;
  static SmemOptIn opt_in;
  if (const int rc = opt_in(kernel, smem, true))
    return rc;
  // In how many parts a sequence's rows are cut: as for chunks (paged_attention_chunk.cu), in blocks of a CTA
  static ClusterFit fit;
  const long long items = (long long)tiles * g.hkv * s.batch;
  const long long seen = std::min<long long>((long long)a.window + a.first + s.max_new, max_rows ? max_rows : s.table_rows);
  const long long blocks = (seen + PD_KEYS - 1) / PD_KEYS;
  int parts = 1;
  long long least = 0;
  for (int p = 1; p <= 16 && blocks >= 2 * W * p; p *= 2) {
    const int at_once = p == 1 ? (W == 4 ? 2 : 1) * sm_count() : fit(kernel, p, W * 32, smem);
    if (at_once <= 0)
      break;
    const long long time = (items + at_once - 1) / at_once * ((blocks + p - 1) / p + (p > 1 ? 12 : 8));
    if (p == 1 || time < least) {
      least = time;
      parts = p;
    }
  }
  // No more CTAs than SMs: one with more warps has more rows on their way. (One stream of 32768 rows, 8 kv heads of 128: 52 us with four warps.)
  if constexpr (W == 4)
    if (items * parts <= sm_count() && blocks >= 4ll * W * parts)
      return launch_few<T, HD, 8>(a, g, s, max_rows, tiles, flags, st);
  cudaLaunchAttribute attr[2];
  cudaLaunchConfig_t cfg = {};
  cfg.attrs = attr;
  cfg.numAttrs = 0;
  if (parts > 1) {
    attr[cfg.numAttrs].id = cudaLaunchAttributeClusterDimension;
    attr[cfg.numAttrs].val.clusterDim.x = parts;
    attr[cfg.numAttrs].val.clusterDim.y = attr[cfg.numAttrs].val.clusterDim.z = 1;
    ++cfg.numAttrs;
  }
  if (flags & NNTR_CUDA_GEMV_PDL) {
    attr[cfg.numAttrs].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[cfg.numAttrs].val.programmaticStreamSerializationAllowed = 1;
    ++cfg.numAttrs;
  }
  cfg.gridDim = dim3((unsigned)(tiles * parts), (unsigned)g.hkv, (unsigned)s.batch);
  cfg.blockDim = dim3(W * 32);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  CUtensorMap maps[2];
  for (int i = 0; i < 2; ++i) {
    const int rc = encode_map_pages(&maps[i], i ? a.v : a.k, g.hd, 1 << g.page_shift, g.hkv, g.n_pages, g.page_stride, PD_KEYS);
    if (rc)
      return rc;
  }
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, maps[0], maps[1], a, g, s);
  count_launch();
  return check_cuda(e, "paged_attention launch");
}

int launch_paged_attention(const nntr_paged_cache *c, const nntr_paged_batch *b, const void *q, int64_t ld_q, unsigned window,
                           unsigned first_tokens, const float *sink, void *out, int out_dtype, int64_t ld_out, unsigned flags,
                           cudaStream_t st) {
  PagedGeom g;
  PagedBatch s;
  int rc = check_paged("paged_attention", c, b, &g, &s);
  if (rc)
    return rc;
  if (s.batch == 0 || s.tokens == 0 || s.max_new == 0)
    return NNTR_CUDA_OK;
  if (!q || !out)
    return set_error(NNTR_CUDA_ERR_INVALID, "paged_attention: null pointer");
  if (out_dtype != c->dtype && out_dtype != NNTR_F32)
    return set_error(NNTR_CUDA_ERR_UNSUPPORTED, "paged_attention: results of the cache's type or fp32 (dtype %d)", out_dtype);
  const int64_t width = (int64_t)g.hq * g.hd;
  if (ld_q < width || ld_q % 8 || (reinterpret_cast<uintptr_t>(q) & 15) || ld_out < width || ld_out % 8 || (reinterpret_cast<uintptr_t>(out) & 15))
    return set_error(NNTR_CUDA_ERR_INVALID, "paged_attention: rows of %lld elements, %lld and %lld apart; need 16-byte aligned rows that do not overlap",
                     (long long)width, (long long)ld_q, (long long)ld_out);
  if (window == 0)
    return set_error(NNTR_CUDA_ERR_INVALID, "paged_attention: a window of no rows");
  constexpr int NONE = 0x3fffffff;
  AttendArgs a = {q, c->kcache, c->vcache, out, sink, ld_q, ld_out, (int)std::min(window, (unsigned)NONE),
                  (int)std::min(first_tokens, (unsigned)NONE), out_dtype == NNTR_F32, LOG2E / sqrtf((float)g.hd)};
  // Up to 32 rows of a kv head's group take the kernel above: its tiles of 16 read the cache twice, the second time from L2, but the other one's
  // steps of 128 rows cost the same for one query row as for 128 (4 x 8000 rows of cache, 8 kv heads of 128: 20 query rows 31.5 and 40.5
  // us, 36 rows 56 and 41). Up to 64 where few CTAs are busy anyway (1 x 8000: 64 rows 19.4 and 23.8; 128 rows 30.5 and 25.2).
  const long long rows = (long long)s.max_new * (g.hq / g.hkv);
  const int tiles = (int)((rows + 15) / 16);
  if (rows > 32 && (rows > 64 || (long long)tiles * g.hkv * s.batch > sm_count() / 4))
    return launch_paged_attention_chunk(a, c->dtype, g, s, b->max_rows, flags, st);
  if (c->dtype == NNTR_F16)
    return g.hd <= 64 ? launch_few<__half, 64, 4>(a, g, s, b->max_rows, tiles, flags, st) : launch_few<__half, 128, 4>(a, g, s, b->max_rows, tiles, flags, st);
  return g.hd <= 64 ? launch_few<__nv_bfloat16, 64, 4>(a, g, s, b->max_rows, tiles, flags, st)
                    : launch_few<__nv_bfloat16, 128, 4>(a, g, s, b->max_rows, tiles, flags, st);
}

} // namespace nntr
