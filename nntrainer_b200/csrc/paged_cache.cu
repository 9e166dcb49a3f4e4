// SPDX-License-Identifier: Apache-2.0
/**
 * @file  paged_cache.cu
 * @brief What writes a key/value cache in pages: the new rows of a batch of sequences (with the per-head norms and the position
 *        rotation of queries and keys), and copies of whole pages.
 *
 * The mathematics of the first is that of MHACoreLayer for one sequence and a contiguous cache
 * (Applications/CausalLM/layers/mha_core.cpp:489-506, reshaped_rms_norm.cpp:84-100):
 *   r = x / sqrt(mean(x^2) + eps) * gamma,   y[i] = r[i] cos - r[i + h] sin,   y[i + h] = r[i] sin + r[i + h] cos,   h = head_dim / 2
 * in fp32, rounded once to the cache's type. Both move bytes and compute next to nothing.
 */
#include "paged.cuh"

#include <algorithm>

namespace nntr {

__device__ int g_paged_cache_status = 0;

int read_paged_cache_status(int *out, bool clear) {
  int v = 0;
  NNTR_CHECK_CUDA(cudaMemcpyFromSymbol(&v, g_paged_cache_status, sizeof(int)));
  if (v && clear) {
    const int zero = 0;
    NNTR_CHECK_CUDA(cudaMemcpyToSymbol(g_paged_cache_status, &zero, sizeof(int)));
  }
  *out = v;
  return NNTR_CUDA_OK;
}

int check_paged(const char *what, const nntr_paged_cache *c, const nntr_paged_batch *b, PagedGeom *g, PagedBatch *s) {
  if (!c || !b || !c->kcache || !c->vcache)
    return set_error(NNTR_CUDA_ERR_INVALID, "%s: null pointer", what);
  if (c->dtype != NNTR_F16 && c->dtype != NNTR_BF16)
    return set_error(NNTR_CUDA_ERR_UNSUPPORTED, "%s: caches of fp16 or bf16 (dtype %d)", what, c->dtype);
  if (!c->n_heads_q || !c->n_heads_kv || c->n_heads_q % c->n_heads_kv || c->n_heads_q > 4096)
    return set_error(NNTR_CUDA_ERR_INVALID, "%s: %u query heads on %u kv heads", what, c->n_heads_q, c->n_heads_kv);
  if (c->head_dim == 0 || c->head_dim % 8)
    return set_error(NNTR_CUDA_ERR_INVALID, "%s: need head_dim %% 8 == 0 (head_dim=%u)", what, c->head_dim);
  if (c->head_dim > 128)
    return set_error(NNTR_CUDA_ERR_UNSUPPORTED, "%s: heads of at most 128 dimensions (head_dim=%u)", what, c->head_dim);
  if (c->page_size < 16 || c->page_size > 256 || (c->page_size & (c->page_size - 1)))
    return set_error(NNTR_CUDA_ERR_UNSUPPORTED, "%s: pages of 16, 32, 64, 128 or 256 rows (page_size=%u)", what, c->page_size);
  const int64_t dense = (int64_t)c->page_size * c->n_heads_kv * c->head_dim, stride = c->page_stride ? c->page_stride : dense;
  if (stride < dense || stride % 8 || (reinterpret_cast<uintptr_t>(c->kcache) & 15) || (reinterpret_cast<uintptr_t>(c->vcache) & 15))
    return set_error(NNTR_CUDA_ERR_INVALID, "%s: pages %lld elements apart, of %lld; need 16-byte aligned pages that do not overlap", what,
                     (long long)stride, (long long)dense);
  if (c->n_pages == 0 || c->n_pages > 0x7fffffffu)
    return set_error(NNTR_CUDA_ERR_INVALID, "%s: a pool of %u pages", what, c->n_pages);
  if (b->batch > 65535 || b->tokens > 0x40000000u / c->n_heads_q || b->max_new > b->tokens)
    return set_error(NNTR_CUDA_ERR_INVALID, "%s: batch of %u sequences, %u rows, %u of them of one sequence", what, b->batch, b->tokens,
                     b->max_new);
  if (b->ld_table > 0x20000000u / c->page_size) // positions and differences of them stay in 32 bits
    return set_error(NNTR_CUDA_ERR_INVALID, "%s: a page table of %u entries per sequence; contexts of at most 2^29 rows", what, b->ld_table);
  if (b->batch && (!b->row_start || !b->context || (b->ld_table && !b->page_table)))
    return set_error(NNTR_CUDA_ERR_INVALID, "%s: null pointer", what);
  int shift = 0;
  while (1u << shift < c->page_size)
    ++shift;
  *g = {(long long)stride, shift, (int)c->n_pages, (int)c->n_heads_q, (int)c->n_heads_kv, (int)c->head_dim};
  *s = {b->row_start, b->context, b->page_table, (int)b->batch, (int)b->tokens, (int)b->max_new, (int)b->ld_table,
        (int)(b->ld_table * c->page_size)};
  return NNTR_CUDA_OK;
}

/* ------------------------------------------------------------- new rows */

constexpr int PA_THREADS = 256;
constexpr int PA_LANES = 16; // of a head: four pairs (i, i + head_dim / 2) each, 16-byte loads
constexpr int PA_HEADS = PA_THREADS / PA_LANES;

struct AppendArgs {
  const float *q, *k, *v, *q_gamma, *k_gamma, *cos_tab, *sin_tab;
  void *q_out, *kcache, *vcache;
  long long ld_q, ld_kv, ld_out;
  float eps;
  int table_rows, chunks, ctas; // chunks: CTAs of a token; ctas: ranges of tokens. One more CTA tells of sequences that contradict the bounds
};

__device__ __forceinline__ float4 load4(const float *p, bool vec) {
  return vec ? *reinterpret_cast<const float4 *>(p) : make_float4(p[0], p[1], p[2], p[3]);
}
template <typename T> __device__ __forceinline__ void store4(T *p, const float4 &f) {
  *reinterpret_cast<uint2 *>(p) = make_uint2(pack2<T>(f.x, f.y), pack2<T>(f.z, f.w));
}

/* A CTA takes 16 U heads (query heads, then key heads, then value heads) of tokens that follow each other, 16 lanes a head, each lane group U
 * heads whose loads are on their way together, before it is looked up where the token belongs. Many tokens are bound by bandwidth, if only
 * few instructions go into an element: what a head's lanes need to know of it is computed once, mean and root by a multiplication and the
 * approximate reciprocal root (2^-22). VEC: rows, gammas and tables are 16-byte aligned.
 * 3760 tokens of 32 + 2 x 8 heads of 128 (139 MB beside the tables): 30.3 us, 4.6 TB/s; one head a lane group, CTAs by heads and
 * divisions 36.2. What is left is waiting: a lane group asks for a token's rows when it is through with the one in front (issue slots 63 %, HBM
 * 45 %). 64 tokens: 3.3 us, the latency of a launch, of one head's loads and of its sum. */
template <typename T, int U, bool VEC>
__global__ void __launch_bounds__(PA_THREADS, U == 1 ? 5 : 4) paged_append_kernel(AppendArgs a, PagedGeom g, PagedBatch s) {
  pdl_launch_dependents();
  const int lane = threadIdx.x & 31, l = threadIdx.x % PA_LANES;
  const int ctas = a.ctas, cta = blockIdx.x / a.chunks, head0 = (blockIdx.x % a.chunks) * (PA_HEADS * U) + threadIdx.x / PA_LANES;
  const int half = g.hd / 2, e = 4 * l;
  const float *src[U], *gamma[U];
  T *to[U]; // row 0 of the caches or of the result
  long long ld[U];
  bool turned[U], query[U], on[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int head = head0 + u * PA_HEADS;
    query[u] = head < g.hq;
    turned[u] = head < g.hq + g.hkv;
    on[u] = head < g.hq + 2 * g.hkv && e < half;
    const int off = (query[u] ? head : turned[u] ? head - g.hq : head - g.hq - g.hkv) * g.hd + e;
    src[u] = (query[u] ? a.q : turned[u] ? a.k : a.v) + off;
    to[u] = static_cast<T *>(query[u] ? a.q_out : turned[u] ? a.kcache : a.vcache) + off;
    gamma[u] = query[u] ? a.q_gamma : a.k_gamma;
    ld[u] = query[u] ? a.ld_q : a.ld_kv;
  }
  const float per_dim = 1.0f / (float)g.hd;
  pdl_wait();
  if (cta >= ctas) { // those too that no token belongs to
    for (int b = threadIdx.x; b < s.batch; b += PA_THREADS)
      if (seq_rows(s, b).bad)
        atomicExch(&g_paged_cache_status, NNTR_CUDA_ERR_INVALID);
    return;
  }
  int seq = 0;
  SeqRows r = {0, 0, 0, false};
  const int last = (int)((long long)s.tokens * (cta + 1) / ctas);
  for (int token = (int)((long long)s.tokens * cta / ctas); token < last; ++token) {
    float4 x[U], y[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      x[u] = y[u] = make_float4(0.f, 0.f, 0.f, 0.f);
      if (on[u]) {
        const float *p = src[u] + token * ld[u];
        x[u] = load4(p, VEC);
        y[u] = load4(p + half, VEC);
      }
    }
    if (token >= r.first + r.n) { // another sequence than the token's in front
      seq = seq_of_row(s, token, lane);
      if (seq >= s.batch)
        return; // behind the last sequence: left as it is
      r = seq_rows(s, seq);
    }
    const int i = token - r.first, pos = r.pos + i;
    if (i < 0 || i >= r.n)
      continue;
    const bool placed = pos >= 0 && pos < a.table_rows; // a row of the rotation tables
    const long long row = placed ? g.row_offset(s, seq, pos, 0) : -1;
    float4 c = make_float4(0.f, 0.f, 0.f, 0.f), n = c; // no rotation is known: the query is zero, no row is stored
    if (placed && e < half) {
      c = load4(a.cos_tab + (size_t)pos * g.hd + e, VEC);
      n = load4(a.sin_tab + (size_t)pos * g.hd + e, VEC);
    }
    if (row < 0 && l == 0)
      atomicExch(&g_paged_cache_status, NNTR_CUDA_ERR_INVALID);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (a.q_gamma) { // all lanes, whatever their heads are: a sum over lanes that not all of a warp may come to costs as much again
        float sum = x[u].x * x[u].x + x[u].y * x[u].y + x[u].z * x[u].z + x[u].w * x[u].w +
                    (y[u].x * y[u].x + y[u].y * y[u].y + y[u].z * y[u].z + y[u].w * y[u].w);
#pragma unroll
        for (int o = PA_LANES / 2; o; o >>= 1)
          sum += __shfl_xor_sync(FULL, sum, o);
        if (turned[u] && on[u]) {
          const float scale = rsqrtf(fmaf(sum, per_dim, a.eps));
          const float4 gx = load4(gamma[u] + e, VEC), gy = load4(gamma[u] + half + e, VEC);
          x[u] = make_float4(x[u].x * scale * gx.x, x[u].y * scale * gx.y, x[u].z * scale * gx.z, x[u].w * scale * gx.w);
          y[u] = make_float4(y[u].x * scale * gy.x, y[u].y * scale * gy.y, y[u].z * scale * gy.z, y[u].w * scale * gy.w);
        }
      }
      if (turned[u]) {
        const float4 p = x[u], t = y[u];
        x[u] = make_float4(p.x * c.x - t.x * n.x, p.y * c.y - t.y * n.y, p.z * c.z - t.z * n.z, p.w * c.w - t.w * n.w);
        y[u] = make_float4(p.x * n.x + t.x * c.x, p.y * n.y + t.y * c.y, p.z * n.z + t.z * c.z, p.w * n.w + t.w * c.w);
      }
      if (on[u] && (query[u] || row >= 0)) {
        T *dst = to[u] + (query[u] ? token * a.ld_out : row);
        store4(dst, x[u]);
        store4(dst + half, y[u]);
      }
    }
  }
}

static void launch_cfg(cudaLaunchConfig_t &cfg, cudaLaunchAttribute *attr, unsigned flags, cudaStream_t st) {
  cfg.stream = st;
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = (flags & NNTR_CUDA_GEMV_PDL) ? 1 : 0;
}

int launch_paged_append(const nntr_paged_cache *c, const nntr_paged_batch *b, const float *q, const float *k, const float *v,
                        int64_t ld_q, int64_t ld_kv, const float *q_gamma, const float *k_gamma, float eps, const float *cos_tab,
                        const float *sin_tab, unsigned table_rows, void *q_out, int64_t ld_out, unsigned flags, cudaStream_t st) {
  PagedGeom g;
  PagedBatch s;
  int rc = check_paged("paged_append", c, b, &g, &s);
  if (rc)
    return rc;
  if (s.batch == 0 || s.tokens == 0)
    return NNTR_CUDA_OK;
  if (!q || !k || !v || !cos_tab || !sin_tab || !q_out)
    return set_error(NNTR_CUDA_ERR_INVALID, "paged_append: null pointer");
  if ((q_gamma == nullptr) != (k_gamma == nullptr))
    return set_error(NNTR_CUDA_ERR_INVALID, "paged_append: q_gamma and k_gamma come together or not at all");
  if (ld_q < (int64_t)g.hq * g.hd || ld_kv < (int64_t)g.hkv * g.hd || ld_out < (int64_t)g.hq * g.hd || ld_out % 4 ||
      (reinterpret_cast<uintptr_t>(q_out) & 7))
    return set_error(NNTR_CUDA_ERR_INVALID, "paged_append: rows %lld, %lld and %lld elements apart; rows must not overlap, those of the result must be 8-byte aligned",
                     (long long)ld_q, (long long)ld_kv, (long long)ld_out);
  if (table_rows > 0x7fffffffu)
    table_rows = 0x7fffffffu;
  AppendArgs a = {q, k, v, q_gamma, k_gamma, cos_tab, sin_tab, q_out, c->kcache, c->vcache, ld_q, ld_kv, ld_out, eps, (int)table_rows, 0, 0};
  uintptr_t low = 0;
  for (const float *p : {q, k, v, q_gamma, k_gamma, cos_tab, sin_tab})
    low |= reinterpret_cast<uintptr_t>(p);
  const bool vec = !(low & 15) && ld_q % 4 == 0 && ld_kv % 4 == 0;
  // Heads of a lane group: one while that many CTAs do not fill the machine twice. CTAs: no more than run at a time, each with tokens
  // that follow each other, which mostly belong to one sequence.
  const int groups = (g.hq + 2 * g.hkv + PA_HEADS - 1) / PA_HEADS;
  const int each = (long long)s.tokens * groups < 16ll * sm_count() ? 1 : groups % 3 == 0 || groups > 4 ? 3 : groups % 2 == 0 ? 2 : groups;
  a.chunks = (groups + each - 1) / each;
  const int at_once = (each == 1 ? 5 : 4) * sm_count() - 1;
  a.ctas = std::min(s.tokens, std::max(1, at_once / a.chunks));
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[1];
  launch_cfg(cfg, attr, flags, st);
  cfg.gridDim = dim3((unsigned)(a.ctas * a.chunks + 1));
  cfg.blockDim = dim3(PA_THREADS);
  auto launch = [&](auto value) {
    using T = decltype(value);
    if (!vec)
      return cudaLaunchKernelEx(&cfg, each == 1 ? paged_append_kernel<T, 1, false> : each == 2 ? paged_append_kernel<T, 2, false> : paged_append_kernel<T, 3, false>, a, g, s);
    return cudaLaunchKernelEx(&cfg, each == 1 ? paged_append_kernel<T, 1, true> : each == 2 ? paged_append_kernel<T, 2, true> : paged_append_kernel<T, 3, true>, a, g, s);
  };
  const cudaError_t e = c->dtype == NNTR_F16 ? launch(__half()) : launch(__nv_bfloat16());
  count_launch();
  return check_cuda(e, "paged_append launch");
}

/* ---------------------------------------------------------- whole pages */

constexpr int CP_THREADS = 256;
constexpr int CP_AT = 4; // 16-byte loads of a thread on their way at a time

/* grid: (pieces of a page, pairs, arrays). Bandwidth bounds it: 16 KB in flight a CTA, eight CTAs on an SM. 133 pages of 64 KB in 48 arrays
 * (837 MB moved): 107 us, a part of it from L2; 3 of 32 KB in 72 arrays 2.6 us, a launch. */
__global__ void __launch_bounds__(CP_THREADS)
copy_pages_kernel(uint8_t *__restrict__ base, long long array_bytes, long long page_bytes, int n_pages, const int *__restrict__ src,
                  const int *__restrict__ dst) {
  pdl_launch_dependents();
  pdl_wait();
  const int from = __ldg(src + blockIdx.y), to = __ldg(dst + blockIdx.y);
  if ((unsigned)from >= (unsigned)n_pages || (unsigned)to >= (unsigned)n_pages) {
    if (threadIdx.x == 0)
      atomicExch(&g_paged_cache_status, NNTR_CUDA_ERR_INVALID);
    return;
  }
  uint8_t *array = base + blockIdx.z * array_bytes;
  const uint4 *a = reinterpret_cast<const uint4 *>(array + from * page_bytes);
  uint4 *d = reinterpret_cast<uint4 *>(array + to * page_bytes);
  const int n = (int)(page_bytes / 16), i0 = blockIdx.x * (CP_THREADS * CP_AT) + threadIdx.x;
  uint4 w[CP_AT];
#pragma unroll
  for (int k = 0; k < CP_AT; ++k)
    if (i0 + k * CP_THREADS < n)
      w[k] = __ldcs(a + i0 + k * CP_THREADS);
#pragma unroll
  for (int k = 0; k < CP_AT; ++k)
    if (i0 + k * CP_THREADS < n)
      __stcs(d + i0 + k * CP_THREADS, w[k]);
}

int launch_copy_pages(void *base, unsigned arrays, int64_t array_bytes, int64_t page_bytes, unsigned n_pages, const int *src,
                      const int *dst, unsigned n, unsigned flags, cudaStream_t st) {
  if (n == 0 || arrays == 0)
    return NNTR_CUDA_OK;
  if (!base || !src || !dst)
    return set_error(NNTR_CUDA_ERR_INVALID, "copy_pages: null pointer");
  if (page_bytes <= 0 || page_bytes % 16 || page_bytes > 0x40000000ll || (reinterpret_cast<uintptr_t>(base) & 15) || array_bytes % 16 ||
      n_pages == 0 || n_pages > 0x7fffffffu || (arrays > 1 && array_bytes < page_bytes * n_pages))
    return set_error(NNTR_CUDA_ERR_INVALID, "copy_pages: %u arrays of %u pages of %lld bytes, %lld bytes apart; need 16-byte aligned pages", arrays,
                     n_pages, (long long)page_bytes, (long long)array_bytes);
  if (n > 65535 || arrays > 65535)
    return set_error(NNTR_CUDA_ERR_UNSUPPORTED, "copy_pages: at most 65535 pairs and arrays per call");
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[1];
  launch_cfg(cfg, attr, flags, st);
  const int64_t piece = 16ll * CP_THREADS * CP_AT;
  cfg.gridDim = dim3((unsigned)((page_bytes + piece - 1) / piece), n, arrays);
  cfg.blockDim = dim3(CP_THREADS);
  const cudaError_t e = cudaLaunchKernelEx(&cfg, copy_pages_kernel, static_cast<uint8_t *>(base), (long long)array_bytes,
                                           (long long)page_bytes, (int)n_pages, src, dst);
  count_launch();
  return check_cuda(e, "copy_pages launch");
}

} // namespace nntr
