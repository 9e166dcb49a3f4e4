// SPDX-License-Identifier: Apache-2.0
/**
 * @file  paged_attention_chunk.cu
 * @brief Attention of chunks of new tokens over a key/value cache in pages, on the tensor cores (tcgen05, kind::f16).
 *
 * The formulas are those of paged_attention.cu. A tile is 128 rows of (token, query head of one kv head's group); a CTA holds two of
 * them against the same cache rows, in steps of 128:
 *   warps 0-7, 8-15 two threads per row of the first / second tile, one half of the step's rows each: S from tensor memory, probabilities
 *                   back over it as the next product's 16-bit operand, their sum. O is multiplied in place only where a row's probabilities
 *                   would outgrow their type with the maximum that they refer to.
 *   warps 16, 17    one for each tile; a thread issues S = Q K^T (both operands in shared memory) and O += P V (P in tensor memory, V as
 *                   it lies, dimensions contiguous). While one tile's probabilities are computed the other tile's products run.
 *   warp 18         TMA copies of K and V tiles through one ring of slots: a box per page (128 rows of it at most) and 64 dimensions.
 *   warp 19         tells of pages and lengths that contradict the bounds.
 * Tensor memory: S (P) 128 columns a tile, O head_dim columns a tile.
 * Few tiles: the CTAs of a cluster share a pair of tiles along the cache rows and join through each other's shared memory.
 * Every wait is bounded (pipeline.cuh).
 *
 * What bounds it. A step's products take 2 * 1024 clocks at head_dim 128, its 2 * 16384 exponentials as many on the special function unit
 * alone (16 a clock). A tile goes round in about 2800: 1400 from its scores to its probabilities (900 of them exponentials of two warps
 * per scheduler), 1030 its products, the rest hand-overs; two tiles overlap. 2 x 2048 tokens of 32 heads of 128 on 8 kv heads at up
 * to 16384 rows: 852 us, 1033 TFLOP/s, at the power limit when it runs for long (1.67 GHz, 990 W). On the way there: 1185
 * with all exponentials on the special function unit, a maximum in every step and both tiles' products issued by one thread; 1024 with
 * exponentials on two units; 960 with the products in turn (TURN_BAR), operands in uniform registers and maxima where a sum asks for them;
 * 890 with two threads per row (a warp alone on its scheduler waits for its own instructions); the masks out of the step's way 852.
 */
#include "cluster.cuh"
#include "paged_attention.cuh"
#include "pipeline.cuh"
#include "tma_map.cuh"

#include <algorithm>

namespace nntr {

__device__ int g_paged_chunk_status = 0;

int read_paged_chunk_status(int *out, bool clear) {
  int v = 0;
  NNTR_CHECK_CUDA(cudaMemcpyFromSymbol(&v, g_paged_chunk_status, sizeof(int)));
  if (v && clear) {
    const int zero = 0;
    NNTR_CHECK_CUDA(cudaMemcpyToSymbol(g_paged_chunk_status, &zero, sizeof(int)));
  }
  *out = v;
  return NNTR_CUDA_OK;
}

namespace {

constexpr int PC_ROWS = 128; // of a tile: the MMA's M, lanes of tensor memory
constexpr int PC_KEYS = 128; // cache rows of a step
constexpr int PC_ROW_WARPS = 8; // of a tile: two threads per row, each with one half of a step's cache rows
constexpr int PC_MMA_WARP = 2 * PC_ROW_WARPS, PC_COPY_WARP = PC_MMA_WARP + 2;
constexpr int PC_THREADS = (PC_MMA_WARP + 4) * 32;
/* Registers of a thread: 96 at launch (640 * 96 of the 65536); the last group gives some to the others: 4 * 104 + 64 = 5 * 96. */
constexpr int PC_REGS_ROWS = 104, PC_REGS_REST = 64;
constexpr uint32_t PC_POLLS = 1u << 22;
template <int HD> struct PcCfg {
  static constexpr int TILE = 128 * HD * 2; // bytes of a tile of Q, K or V: [64 dimensions of HD][row][128 B], 128-byte swizzle
  static constexpr int SLOTS = HD == 128 ? 5 : 8;
  static constexpr int OFF_RING = 2 * TILE;
  static constexpr int OFF_BARS = OFF_RING + SLOTS * TILE;
  static constexpr int OFF_PAIR = OFF_BARS + 256; // a number of each row thread for the row's other one
  static constexpr int OFF_WORK = OFF_PAIR + 2 * 2 * PC_ROWS * 4;
  static constexpr int SMEM = OFF_WORK + 64;
  // a CTA's part of a shared pair of tiles, in the tiles' place
  static constexpr int PITCH = HD + 4; // floats of a row: neighbours' 16-byte pieces fall into different banks
  static constexpr int OFF_ML = 2 * PC_ROWS * PITCH * 4;
  static_assert(OFF_ML + 2 * PC_ROWS * 8 <= OFF_BARS && SMEM <= 227 * 1024, "shared memory of a CTA");
};

__device__ __forceinline__ bool pc_wait(uint32_t bar, uint32_t parity, volatile int *abort_flag) {
  return mbar_wait_warp(bar, parity, abort_flag, &g_paged_chunk_status, PC_POLLS, 2048);
}

/* shared-memory operand in 128-byte swizzled atoms of 8 rows; sbo: from 8 rows to the next 8, lbo: from 64 elements of a row to the next
 * (used where the rows are the K dimension) */
__device__ __forceinline__ uint64_t sw128_desc(uint32_t saddr, uint32_t lbo, uint32_t sbo) {
  return (uint64_t)((saddr >> 4) & 0x3fff) | ((uint64_t)((lbo >> 4) & 0x3fff) << 16) | ((uint64_t)((sbo >> 4) & 0x3fff) << 32) |
         ((uint64_t)1 << 46) | ((uint64_t)2 << 61);
}
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %4, 0;\n\t"
               "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
               : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %4, 0;\n\t"
               "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"(accumulate)
               : "memory");
}
__device__ __forceinline__ void mma_commit(uint32_t bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void tmem_ld32(uint32_t taddr, uint32_t *r) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 "
               "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
                 "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]),
                 "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]),
                 "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
               : "r"(taddr));
}
__device__ __forceinline__ void tmem_st32(uint32_t taddr, const uint32_t *r) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x32.b32 [%32], "
               "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31};" ::"r"(r[0]),
               "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]),
               "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]),
               "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31]), "r"(taddr)
               : "memory");
}
__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint32_t *r) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
                 "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
               : "r"(taddr));
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t *r) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15};" ::"r"(r[0]), "r"(r[1]),
               "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]),
               "r"(r[14]), "r"(r[15]), "r"(taddr)
               : "memory");
}
__device__ __forceinline__ void tmem_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }

template <typename T> struct MmaType;
template <> struct MmaType<__half> {
  static constexpr uint32_t bits = 0;
};
template <> struct MmaType<__nv_bfloat16> {
  static constexpr uint32_t bits = 1u << 7 | 1u << 10;
};

__device__ __forceinline__ float max3(float a, float b, float c) { // NaN if one of them is
  float d;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}

__device__ __forceinline__ float fma_sat(float a, float b, float c) { // a b + c cut to 0 .. 1; NaN: 0
  float d;
  asm("fma.rn.sat.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}

/* 32 scores of a row to probabilities 2^x, x = s * scale - base, packed, and their sum. Some of the pairs are computed on the FMA pipes
 * beside the special function unit, which alone would take as many clocks as a step's products: (UPTO - x) / (UPTO - FROM) cut to 0 .. 1
 * (a power of two: nothing is rounded on the way back; the cut value is to 2^-25, x to 2^-19, in bf16 2^-18), x = n + f with f in
 * [-1/2, 1/2] (the low bits of x + 1.5 * 2^23 are n), 2^f by the polynomial of the least greatest relative error with value 1 at 0 (fp16:
 * fourth degree, 2^-18.4; bf16: third, 2^-13.2), n into the exponent.
 * The cut is what keeps n inside it: in a step that goes by an older maximum x may be anything. It costs nothing where clamping x from below and
 * above took 2.4 % of the long chunks' time and a vote on the greatest x 5 %. What is masked is -inf: zero at FROM, also in bf16 (2^-127
 * has the exponent 0 and no mantissa). */
constexpr int PC_GROUP = 8, PC_BY_FMA = 3; // pairs that go step by step together, so many of them on the FMA pipes
template <typename T>
__device__ __forceinline__ float weights32(const uint32_t *s, float scale, float base, uint32_t *p) {
  constexpr bool FOUR = MmaType<T>::bits == 0;
  constexpr int N = PC_BY_FMA;
  constexpr float WIDE = Weights<T>::UPTO - Weights<T>::FROM, MAGIC = 12582912.f + Weights<T>::UPTO;
  static_assert(WIDE == 64.f || WIDE == 128.f, "a power of two");
  const float per = scale * (-1.f / WIDE), off = (base + Weights<T>::UPTO) * (1.f / WIDE);
  float2 sum = make_float2(0.f, 0.f);
#pragma unroll
  for (int g = 0; g < 16; g += PC_GROUP) {
    float2 x[PC_GROUP], t[PC_GROUP], f[PC_GROUP], q[PC_GROUP];
#pragma unroll
    for (int i = 0; i < PC_GROUP; ++i) {
      const float s0 = __uint_as_float(s[2 * (g + i)]), s1 = __uint_as_float(s[2 * (g + i) + 1]);
      if (i < N) {
        x[i] = make_float2(fma_sat(s0, per, off), fma_sat(s1, per, off));
      } else {
        x[i] = make_float2(-base, -base);
        fma2(x[i].x, x[i].y, s0, s1, scale, scale);
      }
    }
#pragma unroll
    for (int i = 0; i < N; ++i) {
      t[i] = make_float2(MAGIC, MAGIC);
      fma2(t[i].x, t[i].y, x[i].x, x[i].y, -WIDE, -WIDE);
      const float2 n = add2(t[i].x, t[i].y, -MAGIC, -MAGIC); // less UPTO
      f[i] = make_float2(-n.x, -n.y);
      fma2(f[i].x, f[i].y, x[i].x, x[i].y, -WIDE, -WIDE);
      if constexpr (FOUR) {
        q[i] = make_float2(5.590642467794357e-2f, 5.590642467794357e-2f);
        fma2(q[i].x, q[i].y, f[i].x, f[i].y, 9.582853038422538e-3f, 9.582853038422538e-3f);
        float2 r = make_float2(2.4024098611601802e-1f, 2.4024098611601802e-1f);
        fma2(r.x, r.y, q[i].x, q[i].y, f[i].x, f[i].y);
        q[i] = make_float2(6.931241934031505e-1f, 6.931241934031505e-1f);
        fma2(q[i].x, q[i].y, r.x, r.y, f[i].x, f[i].y);
      } else {
        float2 r = make_float2(2.422109594702074e-1f, 2.422109594702074e-1f);
        fma2(r.x, r.y, f[i].x, f[i].y, 5.5008930492411165e-2f, 5.5008930492411165e-2f);
        q[i] = make_float2(6.932829272228233e-1f, 6.932829272228233e-1f);
        fma2(q[i].x, q[i].y, r.x, r.y, f[i].x, f[i].y);
      }
      float2 r = make_float2(1.f, 1.f);
      fma2(r.x, r.y, q[i].x, q[i].y, f[i].x, f[i].y);
      x[i] = make_float2(__uint_as_float(__float_as_uint(r.x) + (__float_as_uint(t[i].x) << 23)),
                         __uint_as_float(__float_as_uint(r.y) + (__float_as_uint(t[i].y) << 23)));
    }
#pragma unroll
    for (int i = N; i < PC_GROUP; ++i)
      x[i] = make_float2(ex2(x[i].x), ex2(x[i].y));
#pragma unroll
    for (int i = 0; i < PC_GROUP; ++i) {
      sum = add2(sum.x, sum.y, x[i].x, x[i].y);
      p[g + i] = pack2<T>(x[i].x, x[i].y);
    }
  }
  return sum.x + sum.y;
}

/* a word whose n lowest bits are set */
__device__ __forceinline__ uint32_t ones_below(int n) { return n <= 0 ? 0u : n >= 32 ? ~0u : (1u << n) - 1; }

/* Barriers of a tile's row threads. They come to every one of them whatever became of their bounded waits: whether one ran out is
 * agreed on here too, and then all leave together. */
__device__ __forceinline__ void rows_sync(int t) {
  asm volatile("barrier.cta.sync %0, %1;" ::"r"(1 + t), "n"(PC_ROW_WARPS * 32) : "memory");
}
__device__ __forceinline__ bool rows_any(int t, bool v) {
  uint32_t r;
  asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %1, 0;\n\tbarrier.cta.red.or.pred q, %2, %3, p;\n\tselp.u32 %0, 1, 0, q;\n\t}"
               : "=r"(r)
               : "r"((uint32_t)v), "r"(1 + t), "n"(PC_ROW_WARPS * 32)
               : "memory");
  return r != 0;
}

/* Pair of tiles number `work` of the batch: its sequence and its place in it, by all lanes of a warp. False: there are fewer. What takes
 * longest comes first, so that it does not begin when the rest is done: in a sequence the last queries, which see most, and among up to
 * 32 sequences those with the longest context. */
__device__ __forceinline__ bool find_pair(const PagedBatch &s, int G, int work, int lane, int *seq, int *tile, SeqRows *r) {
  if (s.batch <= 32) {
    const int b = min(lane, s.batch - 1), lo = __ldg(s.row_start + b), hi = __ldg(s.row_start + b + 1), rows = __ldg(s.context + b);
    const SeqRows own = seq_rows(s, lo, hi, rows);
    const int n = lane < s.batch ? (own.n * G + 2 * PC_ROWS - 1) / (2 * PC_ROWS) : 0;
    int in_front = 0;
    for (int k = 0; k < s.batch; ++k) {
      const int nk = __shfl_sync(FULL, n, k), rk = __shfl_sync(FULL, rows, k);
      in_front += rk > rows || (rk == rows && k < lane) ? nk : 0;
    }
    const unsigned m = __ballot_sync(FULL, work >= in_front && work < in_front + n);
    if (!m)
      return false;
    const int l = __ffs(m) - 1;
    *seq = l;
    *tile = __shfl_sync(FULL, in_front + n - 1 - work, l);
    r->first = __shfl_sync(FULL, own.first, l);
    r->n = __shfl_sync(FULL, own.n, l);
    r->pos = __shfl_sync(FULL, own.pos, l);
    return true;
  }
  int before = 0;
  for (int b0 = 0; b0 < s.batch; b0 += 32) {
    const int n = b0 + lane < s.batch ? (seq_rows(s, b0 + lane).n * G + 2 * PC_ROWS - 1) / (2 * PC_ROWS) : 0;
    int upto = n;
#pragma unroll
    for (int o = 1; o < 32; o *= 2) {
      const int v = __shfl_up_sync(FULL, upto, o);
      upto += lane >= o ? v : 0;
    }
    const unsigned m = __ballot_sync(FULL, before + upto > work);
    if (m) {
      const int l = __ffs(m) - 1;
      *seq = b0 + l;
      *tile = __shfl_sync(FULL, before + upto - 1 - work, l);
      *r = seq_rows(s, *seq);
      return true;
    }
    before += __shfl_sync(FULL, upto, 31);
  }
  return false;
}

} // namespace

template <typename T, int HD>
__global__ void __launch_bounds__(PC_THREADS, 1)
paged_attention_chunk_kernel(const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap, AttendArgs a, PagedGeom g,
                             PagedBatch s) {
  using Cfg = PcCfg<HD>;
  extern __shared__ __align__(1024) uint8_t smem[];
  const uint32_t sbase = smem_u32(smem);
  // numbers that are the same in a warp, and known to be to the compiler: the operands of MMAs are uniform registers
  const int tid = threadIdx.x, warp = __shfl_sync(FULL, tid >> 5, 0), lane = tid & 31;
  const uint32_t bar0 = sbase + Cfg::OFF_BARS;
  // slots full and empty; Q here; of a tile: S complete, P complete, O complete
  auto FULL_BAR = [&](int i) { return bar0 + 8u * i; };
  auto EMPTY_BAR = [&](int i) { return bar0 + 8u * (8 + i); };
  const uint32_t Q_BAR = bar0 + 8 * 16;
  auto S_BAR = [&](int t) { return bar0 + 8u * (17 + t); };
  auto P_BAR = [&](int t) { return bar0 + 8u * (19 + t); };
  auto O_BAR = [&](int t) { return bar0 + 8u * (23 + t); };
  auto TURN_BAR = [&](int t) { return bar0 + 8u * (25 + t); }; // the tile's turn to issue
  uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(smem + Cfg::OFF_BARS + 224);
  volatile int *abort_flag = reinterpret_cast<volatile int *>(smem + Cfg::OFF_BARS + 232);

  if (tid == 32) {
    asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&kmap)));
    asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&vmap)));
  }
  if (tid == 0) {
    for (int i = 0; i < Cfg::SLOTS; ++i) {
      mbar_init(FULL_BAR(i), 1);
      mbar_init(EMPTY_BAR(i), 2); // both tiles
    }
    mbar_init(Q_BAR, 2 * PC_ROW_WARPS);
    for (int t = 0; t < 2; ++t) {
      mbar_init(S_BAR(t), 1);
      mbar_init(P_BAR(t), PC_ROW_WARPS);
      mbar_init(O_BAR(t), 1);
      mbar_init(TURN_BAR(t), 1);
    }
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == PC_MMA_WARP) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(512u) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  fence_before();
  __syncthreads();
  fence_after();
  const uint32_t tmem = __shfl_sync(FULL, *tmem_slot, 0);
  auto S_COL = [&](int t) { return tmem + 128u * t; };
  auto O_COL = [&](int t) { return tmem + 256u + (uint32_t)HD * t; };
  pdl_launch_dependents();
  pdl_wait();

  const int parts = cluster_size(), part = cluster_rank(), G = g.hq / g.hkv, item = blockIdx.x / parts, h = item % g.hkv;
  // What the CTA works on is found by one warp and stays in shared memory: held in registers meanwhile it costs the row threads spills
  volatile int *work = reinterpret_cast<volatile int *>(smem + Cfg::OFF_WORK); // rows, sequence, first row of q, position, place in the group
  if (warp == 0) {
    int seq = 0, tile = 0;
    SeqRows r = {};
    const bool any = find_pair(s, G, item / g.hkv, lane, &seq, &tile, &r); // the same in every CTA of a cluster
    const int flat0 = tile * 2 * PC_ROWS, tok0 = flat0 / G;
    if (lane == 0) {
      work[0] = any ? min(2 * PC_ROWS, r.n * G - flat0) : 0;
      work[1] = seq;
      work[2] = r.first + tok0;
      work[3] = r.pos + tok0;
      work[4] = flat0 - tok0 * G;
    }
  }
  __syncthreads();
  const int rows = work[0], seq = work[1];
  const bool two = rows > PC_ROWS;
  // row k of the pair of tiles: its token, counted from the pair's first one, and its head of the group
  const FastDiv by_g(G);
  auto token_of = [&](int k) { return by_g.div(work[4] + k); };
  auto head_of = [&](int k, int token) { return h * G + work[4] + k - token * G; };
  auto q_row = [&](int token) { return work[2] + token; };
  const Sight sight(work[3], rows > 0 ? work[3] + token_of(rows - 1) : -1, a.window, a.first, PC_KEYS);
  const int b_lo = (int)((long long)sight.blocks * part / parts), steps = (int)((long long)sight.blocks * (part + 1) / parts) - b_lo;

  if (warp >= PC_MMA_WARP)
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(PC_REGS_REST));
  if (warp < PC_MMA_WARP) {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(PC_REGS_ROWS));
    /* ------------------------------ two threads per row ------------------------------ */
    const int t = warp / PC_ROW_WARPS, half = warp / 4 & 1, wrow = (warp & 3) * 32, row = wrow + lane, own = t * PC_ROWS + row;
    const bool there = own < rows;
    const int p = there ? work[3] + token_of(own) : -1;
    constexpr int CH = HD / 8; // 16-byte pieces of a row
    uint4 w[CH / 2]; // 16 rows of the tile, all on their way together
#pragma unroll
    for (int u = 0; u < CH / 2; ++u) {
      const int i = lane + 32 * u, c = i % CH, k = t * PC_ROWS + wrow + 16 * half + i / CH, tok = token_of(k);
      w[u] = make_uint4(0, 0, 0, 0);
      if (k < rows && 8 * c < g.hd)
        w[u] = *reinterpret_cast<const uint4 *>(static_cast<const T *>(a.q) + q_row(tok) * a.ld_q + head_of(k, tok) * g.hd + 8 * c);
    }
#pragma unroll
    for (int u = 0; u < CH / 2; ++u) {
      const int i = lane + 32 * u, c = i % CH, rr = wrow + 16 * half + i / CH;
      sts128(sbase + t * Cfg::TILE + (c >> 3) * (PC_ROWS * 128) + rr * 128 + (((c & 7) ^ (rr & 7)) << 4), w[u].x, w[u].y, w[u].z, w[u].w);
    }
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    __syncwarp();
    if (lane == 0)
      mbar_arrive(Q_BAR);

    const uint32_t trow = (uint32_t)wrow << 16;
    const uint32_t s_at = S_COL(t) + trow + 64 * half, o_at = O_COL(t) + trow + HD / 2 * half; // P begins where the half's scores do
    float *pair_own = reinterpret_cast<float *>(smem + Cfg::OFF_PAIR) + (2 * t + half) * PC_ROWS + row;
    const float *pair_other = reinterpret_cast<const float *>(smem + Cfg::OFF_PAIR) + (2 * t + 1 - half) * PC_ROWS + row;
    float m = -INFINITY, l = 0.f; // the maximum that the row's probabilities refer to, in powers of two; the sum of this half's
    bool ok = true;
    const bool mine = t == 0 ? rows > 0 : two;
    // The scores of step j are complete, and all products issued before them: nobody reads its keys and the values in front of them any
    // more. (An arrival by tcgen05.commit for each slot costs the thread that issues the products time.) Where
    // the second tile has no rows the first gives back for both.
    auto give_back = [&](int j) {
      if (warp % PC_ROW_WARPS == 0 && lane == 0)
        for (int item = max(0, 2 * j - 1); item <= 2 * j; ++item)
          if (item + Cfg::SLOTS < 2 * steps) // nobody waits for a slot that is not filled again
            asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0], %1;" ::"r"(EMPTY_BAR(item % Cfg::SLOTS)), "r"(two ? 1 : 2) : "memory");
    };
    bool unset = true; // a row of the tile has no maximum yet
    for (int j = 0; mine && j < steps; ++j) {
      const bool came = pc_wait(S_BAR(t), j & 1, abort_flag);
      fence_after();
      const int j0 = sight.block(b_lo + j) * PC_KEYS;
      const bool all = j0 + PC_KEYS - 1 <= sight.lo && (j0 > sight.hi - sight.window || j0 + PC_KEYS <= a.first);
      if (!all) { // masked where they are: what follows need not know
#pragma unroll 1
        for (int c = 0; c < 2; ++c) {
          const int k0 = j0 + 64 * half + 32 * c; // bit i: the row sees cache row k0 + i
          const uint32_t seen = ones_below(p + 1 - k0) & (~ones_below(p + 1 - a.window - k0) | ones_below(a.first - k0));
          uint32_t sr[32];
          tmem_ld32(s_at + 32 * c, sr);
          tmem_wait_ld();
#pragma unroll
          for (int i = 0; i < 32; ++i)
            sr[i] = seen >> i & 1 ? sr[i] : 0xff800000u;
          tmem_st32(s_at + 32 * c, sr);
        }
        tmem_wait_st();
      }
      uint32_t pr[32];
      float sum;
      // A row's probabilities refer to a maximum m that is taken in the first step that it sees something of, and where rows are masked. Other
      // steps go by the m there is; what they give shows whether it does. If not the step begins again, with the maximum.
      for (bool afresh = unset || !all;; afresh = true) {
        if (afresh) {
          float mx[2] = {-INFINITY, -INFINITY};
#pragma unroll 1
          for (int c = 0; c < 2; ++c) {
            uint32_t sr[32];
            tmem_ld32(s_at + 32 * c, sr);
            tmem_wait_ld();
#pragma unroll
            for (int i = 0; i < 32; i += 2)
              mx[i >> 1 & 1] = max3(mx[i >> 1 & 1], __uint_as_float(sr[i]), __uint_as_float(sr[i + 1]));
          }
          *pair_own = max3(mx[0], mx[1], mx[1]) * a.scale_log2;
          rows_sync(t);
          float big = max3(*pair_own, *pair_other, *pair_other);
          if (!(big < INFINITY)) { // a score that is no number or infinite: the row's result is NaN, whichever pairs compute its weight
            big = INFINITY;
            l = NAN;
          }
          const bool grown = big > m;
          if (__any_sync(FULL, grown)) {
            const float keep = grown ? ex2(m - big) : 1.f;
            l *= keep;
            if (grown)
              m = big;
            if (j > 0) { // the products so far are complete: S of this step was issued behind them
#pragma unroll
              for (int c = 0; c < HD / 32; ++c) {
                uint32_t o[16];
                tmem_ld16(o_at + 16 * c, o);
                tmem_wait_ld();
#pragma unroll
                for (int i = 0; i < 16; ++i)
                  o[i] = __float_as_uint(__uint_as_float(o[i]) * keep);
                tmem_st16(o_at + 16 * c, o);
              }
            }
          }
          unset = rows_any(t, there && m == -INFINITY);
        }
        const float base = m == -INFINITY ? 0.f : m - Weights<T>::LIFT;
        sum = 0.f;
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          uint32_t sr[32];
          tmem_ld32(s_at + 32 * c, sr);
          tmem_wait_ld();
          sum += weights32<T>(sr, a.scale_log2, base, pr + 16 * c);
        }
        if (!rows_any(t, !came || !(afresh || sum <= Weights<T>::MOST)))
          break;
        if (rows_any(t, !came)) {
          ok = false;
          break;
        }
      }
      if (!ok)
        break;
      tmem_st32(s_at, pr);
      l += sum;
      tmem_wait_st();
      fence_before();
      __syncwarp();
      if (lane == 0)
        mbar_arrive(P_BAR(t));
      give_back(j); // behind what the products wait for
    }

    /* ------------------------------ the row's result ------------------------------ */
    if (mine && steps > 0 && ok)
      ok = pc_wait(O_BAR(t), 0, abort_flag);
    if (two && parts > 1 && steps > 0 && ok) // what follows is written where the other tile's products read
      ok = pc_wait(O_BAR(1 - t), 0, abort_flag);
    fence_after();
    if (mine) {
      *pair_own = l;
      rows_sync(t);
      l += *pair_other;
    }
    if (mine && ok) {
      float inv = 1.f;
      if (parts == 1) {
        float total = l;
        if (a.sink && there)
          total += ex2(a.sink[head_of(own, token_of(own))] * LOG2E - (m - Weights<T>::LIFT));
        inv = m == -INFINITY || total == 0.f ? 0.f : 1.f / total;
      }
      // Rows by threads would be stored as 16 bytes of 32 rows at a time: they go through shared memory, where the tile's queries were, 16-byte
      // pieces spread over the banks; fp32 ones directly.
      const uint32_t turn = sbase + t * Cfg::TILE + row * (HD * 2);
      float *part_row = reinterpret_cast<float *>(smem) + own * Cfg::PITCH;
#pragma unroll
      for (int c = 0; c < HD / 64; ++c) {
        uint32_t o[32];
        if (steps > 0) {
          tmem_ld32(o_at + 32 * c, o);
          tmem_wait_ld();
        } else {
#pragma unroll
          for (int i = 0; i < 32; ++i)
            o[i] = 0u;
        }
#pragma unroll
        for (int i = 0; i < 32; i += 8) {
          float f[8];
#pragma unroll
          for (int k = 0; k < 8; ++k)
            f[k] = __uint_as_float(o[i + k]) * inv;
          const int col = HD / 2 * half + 32 * c + i;
          if (parts > 1) {
            *reinterpret_cast<float4 *>(part_row + col) = make_float4(f[0], f[1], f[2], f[3]);
            *reinterpret_cast<float4 *>(part_row + col + 4) = make_float4(f[4], f[5], f[6], f[7]);
          } else if (!a.out_f32) {
            sts128(turn + ((col >> 3 ^ (row & (HD / 8 - 1))) << 4), pack2<T>(f[0], f[1]), pack2<T>(f[2], f[3]), pack2<T>(f[4], f[5]), pack2<T>(f[6], f[7]));
          } else if (there && col < g.hd) {
            const int token = token_of(own);
            float4 *dst = reinterpret_cast<float4 *>(static_cast<float *>(a.out) + q_row(token) * a.ld_out + head_of(own, token) * g.hd + col);
            dst[0] = make_float4(f[0], f[1], f[2], f[3]);
            dst[1] = make_float4(f[4], f[5], f[6], f[7]);
          }
        }
      }
      if (parts > 1 && half == 0)
        *reinterpret_cast<float2 *>(smem + Cfg::OFF_ML + 8 * own) = make_float2(m, l);
    }
    if (mine && parts == 1 && !a.out_f32) {
      if (!rows_any(t, !ok)) {
#pragma unroll
        for (int u = 0; u < CH / 2; ++u) {
          const int i = lane + 32 * u, c = i % CH, rr = wrow + 16 * half + i / CH, k = t * PC_ROWS + rr, tok = token_of(k);
          const uint4 v = lds128(sbase + t * Cfg::TILE + rr * (HD * 2) + ((c ^ (rr & (CH - 1))) << 4));
          if (k < rows && 8 * c < g.hd)
            *reinterpret_cast<uint4 *>(static_cast<T *>(a.out) + q_row(tok) * a.ld_out + head_of(k, tok) * g.hd + 8 * c) = v;
        }
      }
    }
  } else if (warp < PC_COPY_WARP) {
    /* ------------------------------ products ------------------------------ */
    constexpr uint32_t IDESC = 1u << 4 | MmaType<T>::bits | (uint32_t)(PC_ROWS >> 4) << 24;
    constexpr uint32_t IDESC_S = IDESC | (uint32_t)(PC_KEYS >> 3) << 17;
    constexpr uint32_t IDESC_O = IDESC | (uint32_t)(HD >> 3) << 17 | 1u << 16; // B: its rows are the K dimension
    const int t = warp - PC_MMA_WARP;
    const bool mine = t == 0 || two;
    auto slot_at = [&](int item) { return sbase + Cfg::OFF_RING + (item % Cfg::SLOTS) * Cfg::TILE; };
    auto here = [&](int item) { return pc_wait(FULL_BAR(item % Cfg::SLOTS), item / Cfg::SLOTS & 1, abort_flag); };
    auto scores = [&](int item) {
#pragma unroll
      for (int k = 0; k < HD / 16; ++k) {
        const uint32_t at = (k >> 2) * (128 * 128) + (k & 3) * 32;
        mma_ss(S_COL(t), sw128_desc(sbase + t * Cfg::TILE + at, 0, 1024), sw128_desc(slot_at(item) + at, 0, 1024), IDESC_S, k != 0);
      }
      mma_commit(S_BAR(t));
    };
    // The tiles' products are issued in turn, never mixed: mixed ones are all through at the same time, and then the row threads of both tiles
    // work while the tensor cores wait. Batch n is S of step 0, or O of step n - 1 and S of step n.
    auto my_turn = [&](int n) { return !two || (t == 0 && n == 0) || pc_wait(TURN_BAR(t), (t == 0 ? n - 1 : n) & 1, abort_flag); };
    auto your_turn = [&] {
      if (two)
        mbar_arrive(TURN_BAR(1 - t));
    };
    bool ok = mine && rows > 0 && steps > 0 && pc_wait(Q_BAR, 0, abort_flag) && here(0) && my_turn(0);
    if (ok && elected()) {
      fence_after();
      scores(0);
      your_turn();
    }
    for (int j = 0; j < steps && ok; ++j) {
      const int vi = 2 * j + 1, ki = 2 * j + 2, j0 = sight.block(b_lo + j) * PC_KEYS;
      if (!(ok = here(vi)))
        break;
      if (!(j0 + PC_KEYS - 1 <= sight.hi && (j0 >= sight.from || j0 + PC_KEYS <= sight.first))) {
        // rows that nobody sees meet probabilities of zero: what they hold must be finite (both warps write the same zeros)
        for (int i = lane; i < PC_KEYS * (HD / 8); i += 32) {
          const int rr = i >> 3 & (PC_KEYS - 1);
          if (!sight.row_read(j0 + rr))
            sts128(slot_at(vi) + 16 * i, 0, 0, 0, 0);
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
      }
      if (j + 1 < steps && !(ok = here(ki)))
        break;
      if (!(ok = my_turn(j + 1) && pc_wait(P_BAR(t), j & 1, abort_flag)))
        break;
      fence_after();
      if (elected()) {
#pragma unroll
        for (int k = 0; k < PC_KEYS / 16; ++k)
          mma_ts(O_COL(t), S_COL(t) + 64 * (k >> 2) + 8 * (k & 3), sw128_desc(slot_at(vi) + k * 2048, 128 * 128, 1024), IDESC_O, j != 0 || k != 0);
        if (j + 1 == steps)
          mma_commit(O_BAR(t));
        else
          scores(ki);
        if (t == 0 || j + 1 < steps) // nobody waits for the last one
          your_turn();
      }
    }
    __syncwarp();
  } else if (warp == PC_COPY_WARP) {
    /* ------------------------------ copies ------------------------------ */
    const int page_rows = 1 << g.page_shift, box = min(page_rows, PC_KEYS);
    constexpr int HALVES = HD / 64;
    const int boxes = PC_KEYS / box * HALVES, at_row = lane / HALVES * box, half = lane % HALVES;
    int page = 0, row = 0;
    for (int i = 0; rows > 0 && i < 2 * steps; ++i) {
      if ((i & 1) == 0 && lane < boxes) { // pages of the step, the same for keys and values
        const int at = sight.block(b_lo + i / 2) * PC_KEYS + at_row;
        page = g.n_pages; // outside the map: the box is filled with zeros
        row = at & (page_rows - 1);
        if (at <= sight.hi) {
          const int given = __ldg(s.table + (size_t)seq * s.ld_table + (at >> g.page_shift));
          if ((unsigned)given < (unsigned)g.n_pages)
            page = given;
        }
      }
      const int slot = i % Cfg::SLOTS, use = i / Cfg::SLOTS;
      if (use > 0 && !pc_wait(EMPTY_BAR(slot), (use - 1) & 1, abort_flag))
        break;
      if (lane == 0)
        mbar_expect_tx(FULL_BAR(slot), Cfg::TILE);
      __syncwarp();
      if (lane < boxes)
        tma_box4(sbase + Cfg::OFF_RING + slot * Cfg::TILE + half * (PC_KEYS * 128) + at_row * 128, i & 1 ? &vmap : &kmap, half * 64, row, h, page,
                 FULL_BAR(slot));
    }
    __syncwarp();
  } else {
    /* ------------------------------ contradictions ------------------------------ */
    // Pages outside the pool that a query sees a row of; others may have been given back. Apart from the copies, whose way to a page is short so.
    const int box_shift = min(g.page_shift, 7), each = PC_KEYS >> box_shift;
    for (int i = lane; i < steps * each; i += 32) {
      const int at = sight.block(b_lo + i / each) * PC_KEYS + (i % each << box_shift);
      if (sight.any_read(at, 1 << box_shift) &&
          (unsigned)__ldg(s.table + (size_t)seq * s.ld_table + (at >> g.page_shift)) >= (unsigned)g.n_pages)
        atomicExch(&g_paged_chunk_status, NNTR_CUDA_ERR_INVALID);
    }
    if (blockIdx.x == 0) // a sequence that has no rows has no CTA either
      for (int b = lane; b < s.batch; b += 32)
        if (seq_rows(s, b).bad)
          atomicExch(&g_paged_chunk_status, NNTR_CUDA_ERR_INVALID);
    __syncwarp();
  }

  /* ------------------------------ a shared pair of tiles ------------------------------ */
  if (parts > 1) {
    cluster_sync();
    const uint32_t raised = neighbour_raised(smem_u32(const_cast<int *>(abort_flag)), lane);
    if (warp < PC_MMA_WARP && !__any_sync(FULL, raised)) {
      for (int R = part + parts * warp; R < rows; R += parts * PC_MMA_WARP) {
        const int tok = token_of(R), head = head_of(R, tok), col = 4 * lane;
        float2 ml[8];
        float4 v[8];
#pragma unroll
        for (int k = 0; k < 8; ++k)
          if (k < parts) {
            uint32_t remote;
            asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(sbase + Cfg::OFF_ML + 8 * R), "r"(k));
            asm volatile("ld.shared::cluster.v2.f32 {%0,%1}, [%2];" : "=f"(ml[k].x), "=f"(ml[k].y) : "r"(remote) : "memory");
            v[k] = make_float4(0.f, 0.f, 0.f, 0.f);
            if (col < HD)
              v[k] = ld_cluster4(sbase + 4 * (R * Cfg::PITCH + col), k);
          }
        float big = -INFINITY;
#pragma unroll
        for (int k = 0; k < 8; ++k)
          if (k < parts)
            big = fmaxf(big, ml[k].x);
        float4 f = make_float4(0.f, 0.f, 0.f, 0.f);
        float total = 0.f;
#pragma unroll
        for (int k = 0; k < 8; ++k)
          if (k < parts) {
            const float w = ml[k].x == -INFINITY ? 0.f : ex2(ml[k].x - big);
            total += w * ml[k].y;
            f = make_float4(f.x + w * v[k].x, f.y + w * v[k].y, f.z + w * v[k].z, f.w + w * v[k].w);
          }
        if (a.sink && big > -INFINITY)
          total += ex2(a.sink[head] * LOG2E - (big - Weights<T>::LIFT));
        const float inv = total == 0.f ? 0.f : 1.f / total;
        const long long e = q_row(tok) * a.ld_out + (long long)head * g.hd + col;
        if (col < g.hd) {
          if (a.out_f32)
            *reinterpret_cast<float4 *>(static_cast<float *>(a.out) + e) = make_float4(f.x * inv, f.y * inv, f.z * inv, f.w * inv);
          else
            *reinterpret_cast<uint2 *>(static_cast<T *>(a.out) + e) = make_uint2(pack2<T>(f.x * inv, f.y * inv), pack2<T>(f.z * inv, f.w * inv));
        }
      }
    }
    cluster_sync(); // nobody leaves while its part is read
  }

  /* on an abort copies and products in flight get time to land before the memory is released */
  if (*abort_flag)
    for (int i = 0; i < 1000; ++i)
      __nanosleep(1000);
  fence_before();
  __syncthreads();
  if (warp == PC_MMA_WARP)
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u));
}

/* ------------------------------------------------------------------ launch */

template <typename T, int HD>
static int launch_chunk(const AttendArgs &a, const PagedGeom &g, const PagedBatch &s, unsigned max_rows, unsigned flags, cudaStream_t st) {
  auto kernel = paged_attention_chunk_kernel<T, HD>;
  constexpr int smem = PcCfg<HD>::SMEM;
  static SmemOptIn opt_in;
  if (const int rc = opt_in(kernel, smem))
    return rc;
  CUtensorMap maps[2];
  for (int i = 0; i < 2; ++i) {
    const int rc = encode_map_pages(&maps[i], i ? a.v : a.k, g.hd, 1 << g.page_shift, g.hkv, g.n_pages, g.page_stride,
                                    std::min(1 << g.page_shift, PC_KEYS));
    if (rc)
      return rc;
  }
  const int G = g.hq / g.hkv;
  const long long pair = 2 * PC_ROWS;
  // no sequence has more than max_new rows, and all together no more than `tokens`
  const long long pairs = std::min(s.batch * (((long long)s.max_new * G + pair - 1) / pair), (long long)s.tokens * G / pair + s.batch);
  const long long seen = std::min<long long>((long long)a.window + a.first + s.max_new, max_rows ? max_rows : s.table_rows);
  const long long blocks = (seen + PC_KEYS - 1) / PC_KEYS;
  // In how many parts a pair of tiles is cut, by the steps that the last CTA ends after: waves of as many clusters as run at a time, each
  // of a part's steps and about three more for its start; joining the parts takes about as long as two. (2 x 2048 tokens at up to
  // 16384 rows: 512 pairs on 148 SMs are 4 waves of 120 steps, in two parts 7 of 60.)
  static ClusterFit fit;
  const long long items = pairs * g.hkv;
  int parts = 1;
  long long least = 0;
  for (int p = 1; p <= 8 && blocks >= 2 * p; p *= 2) {
    const int at_once = p == 1 ? sm_count() : fit(kernel, p, PC_THREADS, smem);
    if (at_once <= 0)
      break;
    const long long steps = (items + at_once - 1) / at_once * ((blocks + p - 1) / p + (p > 1 ? 5 : 3));
    if (p == 1 || steps < least) {
      least = steps;
      parts = p;
    }
  }
  cudaLaunchAttribute attr[2];
  cudaLaunchConfig_t cfg = {};
  cfg.attrs = attr;
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
  if (items * parts > 0x7fffffffll)
    return set_error(NNTR_CUDA_ERR_UNSUPPORTED, "paged_attention: too many rows in one call");
  cfg.gridDim = dim3((unsigned)(items * parts));
  cfg.blockDim = dim3(PC_THREADS);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, maps[0], maps[1], a, g, s);
  count_launch();
  return check_cuda(e, "paged_attention launch");
}

int launch_paged_attention_chunk(const AttendArgs &a, int dtype, const PagedGeom &g, const PagedBatch &s, unsigned max_rows, unsigned flags,
                                 cudaStream_t st) {
  if (dtype == NNTR_F16)
    return g.hd <= 64 ? launch_chunk<__half, 64>(a, g, s, max_rows, flags, st) : launch_chunk<__half, 128>(a, g, s, max_rows, flags, st);
  return g.hd <= 64 ? launch_chunk<__nv_bfloat16, 64>(a, g, s, max_rows, flags, st)
                    : launch_chunk<__nv_bfloat16, 128>(a, g, s, max_rows, flags, st);
}

} // namespace nntr
