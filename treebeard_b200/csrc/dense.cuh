// Matrix products on the tensor cores with what follows them fused in:
//   C[m, n] = sum_k A[m, k] B[n, k],  A, B fp16 or bf16, sums in fp32 in tensor memory.
//
// Either operand may lie with k or with its rows one behind the other in memory (the products of the
// backward passes sum over rows): the tensor map's box and the shared-memory descriptor differ, nothing is
// transposed.  A block has one warp that issues the tensor copies, one that issues the matrix instructions
// and sixteen that take finished sums out of tensor memory and, through shared memory, on their way (a chunk of
// theirs is one chain of short steps, so that eight warps took twice as long as sixteen).  Blocks are
// persistent and walk over units: a row tile, a run of column tiles, a part of the sum.
//
// Three shapes (kernel template SHAPE).  Their rates follow what they move through shared memory (128 bytes a cycle),
// which tensor copies write and the matrix unit reads.  With 64 k at a time, bytes written + read per cycle of matrix
// work:
//   kDenseTall  two blocks on 512 x 256 results, 256 rows of A and 128 of B each: 48 + 64.  Both accumulators,
//               128 x 256 a block, belong to one tile; so that one is taken out while the other is still computed,
//               the first runs ahead of the second by up to three stages at a tile's beginning and two at its end.
//   kDensePair  two blocks on 256 x 256 results, 128 rows of each operand: 64 + 64, measured at three quarters of
//               the tall one's rate; two tiles' accumulators, one taken out while the other is computed.
//   kDenseOne   one block on 128 x 128 results, for products with few tiles: 128 + 128, half the rate.
// Plain products, bf16: 8192 x 8192 x 8192 at 1.50 to 1.53 PFLOP/s (cuBLAS 1.60), 32768 x 1024 -> 4096 at 1.35 to 1.39
// (1.40), in 198 to 205 us; with gelu and the value before it as a second result 267 to 316.
// Those bytes are not all: of 4096 x 512 -> 100003 classes (332 to 346 us; the tensor pipe is busy 67 % of the cycles, at
// 1.62 GHz) a pair that kept A in shared memory for eight tiles, 32 + 64, took 31 us more, one with six stages instead of
// four as long as this.
//
// All waits are bounded: one that gives up ends the launch with a word in tb_dense_status.
#pragma once
#include <cuda.h>
#include <cstdint>
#include <type_traits>
#include "element.cuh"
#include "out_pieces.h"

namespace tb {

constexpr int kDenseEndWarps = 16, kDenseThreads = 128 + 32 * kDenseEndWarps, kDenseK = 64;
enum DenseShape { kDenseOne = 0, kDensePair = 1, kDenseTall = 2 };
constexpr int kDenseEndBytes = 4096, kDenseBiasBytes = 256; // a finishing warp's own shared memory
__host__ __device__ constexpr int dense_rows(int shape) { return shape == kDenseTall ? 512 : shape == kDensePair ? 256 : 128; }
__host__ __device__ constexpr int dense_cols(int shape) { return shape == kDenseOne ? 128 : 256; }
__host__ __device__ constexpr int dense_stages(int shape) { return shape == kDenseTall ? 3 : 4; }
__host__ __device__ constexpr int dense_stage_bytes(int shape) { return shape == kDenseTall ? 49152 : 32768; }
__host__ __device__ constexpr int dense_smem_bytes(int shape) {
  return 1024 + dense_stages(shape) * dense_stage_bytes(shape) + kDenseEndWarps * (kDenseEndBytes + kDenseBiasBytes) + 512;
}

__device__ int tb_dense_status; // 0, or 4: a wait gave up

struct DenseProblem {
  CUtensorMap a, b;
  int M, N;
  int a_rows_inner, b_rows_inner; // 1: rows lie one behind the other, not k
  int m_tiles, n_tiles, k_blocks;
  int chunk, chunks; // column tiles of a unit, units along the columns
  int splits;        // parts of the sum
  int group;         // row tiles that are walked together
  int units;
};
// Up to two products of one launch: the second one's units follow the first one's, so that the last wave of one
// and the first of the other share the multiprocessors.
template <class End, int JOBS> struct DenseJobs {
  DenseProblem p[JOBS];
  End end[JOBS];
  int units; // of all
};

__device__ __forceinline__ uint32_t dense_smem(const void *p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void dense_bar_init(uint32_t bar, uint32_t count) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count) : "memory");
}
__device__ __forceinline__ void dense_expect(uint32_t bar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
__device__ __forceinline__ bool dense_try(uint32_t bar, uint32_t parity) {
  uint32_t ok;
  asm volatile("{\n .reg .pred p;\n mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n selp.u32 %0, 1, 0, p;\n}"
               : "=r"(ok) : "r"(bar), "r"(parity) : "memory");
  return ok != 0;
}
// Two seconds at most (a tile takes microseconds).
__device__ __forceinline__ bool dense_wait(uint32_t bar, uint32_t parity) {
  if (dense_try(bar, parity)) return true;
  const long long t0 = clock64();
  for (uint32_t i = 1;; ++i) {
    if (dense_try(bar, parity)) return true;
    if ((i & 63) == 0 && clock64() - t0 > 4000000000ll) return false;
  }
}
// Address of the same shared-memory object in the pair's first block.
__device__ __forceinline__ uint32_t dense_first(uint32_t addr) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(r) : "r"(addr));
  return r;
}
template <bool PAIR>
__device__ __forceinline__ void dense_load(uint32_t dst, const CUtensorMap *map, int x, int y, uint32_t bar) {
  if constexpr (PAIR)
    asm volatile("cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];"
                 ::"r"(dst), "l"(map), "r"(x), "r"(y), "r"(bar) : "memory");
  else
    asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];"
                 ::"r"(dst), "l"(map), "r"(x), "r"(y), "r"(bar) : "memory");
}
template <bool PAIR> __device__ __forceinline__ void dense_commit(uint32_t bar) {
  if constexpr (PAIR)
    asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;"
                 ::"r"(bar), "h"((uint16_t)3) : "memory");
  else
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}
template <bool PAIR>
__device__ __forceinline__ void dense_mma(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t add) {
  if constexpr (PAIR)
    asm volatile("{\n .reg .pred p;\n setp.ne.u32 p, %4, 0;\n"
                 " tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n}" ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(add) : "memory");
  else
    asm volatile("{\n .reg .pred p;\n setp.ne.u32 p, %4, 0;\n"
                 " tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}" ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(add) : "memory");
}
// 32 columns of a warp's 32 rows out of tensor memory; there after dense_taken, which every use depends on.
__device__ __forceinline__ void dense_take(uint32_t addr, uint32_t (&r)[32]) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
               : "r"(addr));
}
__device__ __forceinline__ void dense_taken(uint32_t (&r)[32]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;" : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]), "+r"(r[16]), "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]), "+r"(r[22]), "+r"(r[23]), "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]), "+r"(r[29]), "+r"(r[30]), "+r"(r[31]) :: "memory");
}
// Operand in shared memory, 128-byte swizzle: k one behind the other: 8 rows of 64 k per 1 KB; rows one
// behind the other: 64 rows x 64 k per 8 KB (the leading offset), 8 k per 1 KB.
__device__ __forceinline__ uint64_t dense_desc(uint32_t addr, bool rows_inner) {
  uint64_t d = (uint64_t)((addr & 0x3ffffu) >> 4);
  d |= (uint64_t)(rows_inner ? 8192u >> 4 : 1u) << 16;
  d |= (uint64_t)(1024u >> 4) << 32;
  d |= 1ull << 46; // descriptor version of this architecture
  d |= 2ull << 61; // 128-byte swizzle
  return d;
}
template <class T> __device__ __forceinline__ constexpr uint32_t dense_format();
template <> __device__ __forceinline__ constexpr uint32_t dense_format<__half>() { return 0; }
template <> __device__ __forceinline__ constexpr uint32_t dense_format<__nv_bfloat16>() { return 1; }

struct DenseUnit {
  int m, n0, n1, k0, k1, split, chunk;
};
__device__ __forceinline__ DenseUnit dense_unit(const DenseProblem &p, int u) {
  DenseUnit w;
  int r = u;
  w.split = 0;
  if (p.splits > 1) w.split = u % p.splits, r = u / p.splits;
  const int per = p.group * p.chunks, g = r / per, in = r - g * per, rows = min(p.group, p.m_tiles - g * p.group);
  w.chunk = in / rows;
  w.m = g * p.group + in - w.chunk * rows;
  w.n0 = w.chunk * p.chunk;
  w.n1 = min(w.n0 + p.chunk, p.n_tiles);
  w.k0 = 0, w.k1 = p.k_blocks;
  if (p.splits > 1) {
    w.k0 = (int)((long long)w.split * p.k_blocks / p.splits);
    w.k1 = (int)((long long)(w.split + 1) * p.k_blocks / p.splits);
  }
  return w;
}

// A finishing warp's place: 4 KB and 256 bytes of shared memory, a barrier for copies into it.
struct DenseWarp {
  unsigned char *mine;
  unsigned char *bias;
  uint32_t bar, phase;
  OutPieces out; // of `mine`, 2 KB each
  bool ok, coming; // coming (lane 0): a copy was asked for and has not been waited for
};

// End: what becomes of a tile.  A thread of a finishing warp has one row and 32 columns at a time:
//   start(state, p, row, unit)              once per unit and row
//   tile(p, n, warp)                        once per column tile, n the warp's first column
//   ahead(p, row, n, columns, warp)         before the wait for the sums of these columns
//   chunk(state, p, r, row, n, unit, warp, second, more)   r[j] = C[row, n + j] (bits); row = the warp's first row + lane;
//                                           second: not the warp's first 32 columns; more: 32 more follow
//   stop(state, p, row, unit, part)         after the unit's last tile; part: which quarter of the columns the warp had
template <class T, int SHAPE, class End, int JOBS>
__global__ void __cluster_dims__(SHAPE == kDenseOne ? 1 : 2, 1, 1) __launch_bounds__(kDenseThreads, 1)
    tb_dense_kernel(const __grid_constant__ DenseJobs<End, JOBS> jobs) {
  constexpr bool PAIR = SHAPE != kDenseOne;
  constexpr int BM = dense_rows(SHAPE), BN = dense_cols(SHAPE), MT = SHAPE == kDenseTall ? 2 : 1;
  constexpr int kStages = dense_stages(SHAPE), kStageBytes = dense_stage_bytes(SHAPE), kColumns = BN / 4; // of a finishing warp
  extern __shared__ unsigned char raw[];
  const uint32_t base = (dense_smem(raw) + 1023u) & ~1023u;
  unsigned char *end_p = raw + (base - dense_smem(raw)) + kStages * kStageBytes;
  const uint32_t bars = base + kStages * kStageBytes + kDenseEndWarps * (kDenseEndBytes + kDenseBiasBytes);
  const uint32_t full = bars, empty = bars + 48, tfull = bars + 96, tempty = bars + 112, own = bars + 128, tmem_at = bars + 256;
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const uint32_t rank = PAIR ? blockIdx.x & 1 : 0;
  const int first = PAIR ? blockIdx.x >> 1 : blockIdx.x, step = PAIR ? gridDim.x >> 1 : gridDim.x;
  // f(product, End, unit of it) for the block's u-th unit; the products' fields are constants of each branch
  // (indexed, they would be loads)
  auto of_job = [&](int u, auto f) {
    if constexpr (JOBS == 2) {
      if (u >= jobs.p[0].units) return f(jobs.p[1], jobs.end[1], u - jobs.p[0].units);
    }
    f(jobs.p[0], jobs.end[0], u);
  };

  if (warp == 0 && lane == 0) {
    for (int i = 0; i < kStages; ++i) {
      dense_bar_init(full + 8 * i, 1);
      dense_bar_init(empty + 8 * i, 1);
    }
    for (int i = 0; i < 2; ++i) {
      dense_bar_init(tfull + 8 * i, 1);
      dense_bar_init(tempty + 8 * i, kDenseEndWarps * (PAIR ? 2 : 1));
    }
    for (int i = 0; i < kDenseEndWarps; ++i) dense_bar_init(own + 8 * i, 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 2) {
    if constexpr (PAIR) {
      asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(tmem_at), "r"(2 * BN) : "memory");
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    } else {
      asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(tmem_at), "r"(2 * BN) : "memory");
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  }
  __syncthreads();
  if constexpr (PAIR) {
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
  }
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  uint32_t tmem;
  asm volatile("ld.shared.b32 %0, [%1];" : "=r"(tmem) : "r"(tmem_at));
  after_previous_kernel();

  bool ok = true;
  if (warp == 0) {
    if (lane == 0) {
      int stage = 0;
      uint32_t phase = 0;
      int loads = 0;
      for (int unit = first; ok && unit < jobs.units; unit += step) of_job(unit, [&](const DenseProblem &p, const End &, int u) {
        const DenseUnit w = dense_unit(p, u);
        const int row = w.m * BM + (int)rank * 128;
        for (int n = w.n0; ok && n < w.n1; ++n) {
          const int col = n * BN + (int)rank * 128;
          for (int k = w.k0; k < w.k1; ++k) {
            if (!(ok = dense_wait(empty + 8 * stage, phase ^ 1))) break;
            const uint32_t bar = PAIR ? dense_first(full + 8 * stage) : full + 8 * stage;
            if (rank == 0) dense_expect(full + 8 * stage, kStageBytes * (PAIR ? 2 : 1));
            const uint32_t a = base + stage * kStageBytes, b = a + MT * 16384;
#pragma unroll
            for (int j = 0; j < MT; ++j) {
              if (p.a_rows_inner) {
                dense_load<PAIR>(a + j * 16384, &p.a, row + j * 256, k * kDenseK, bar);
                dense_load<PAIR>(a + j * 16384 + 8192, &p.a, row + j * 256 + 64, k * kDenseK, bar);
              } else {
                dense_load<PAIR>(a + j * 16384, &p.a, k * kDenseK, row + j * 256, bar);
              }
            }
            if (p.b_rows_inner) {
              dense_load<PAIR>(b, &p.b, col, k * kDenseK, bar);
              dense_load<PAIR>(b + 8192, &p.b, col + 64, k * kDenseK, bar);
            } else {
              dense_load<PAIR>(b, &p.b, k * kDenseK, col, bar);
            }
            loads = min(loads + 1, kStages);
            if (++stage == kStages) stage = 0, phase ^= 1;
          }
        }
      });
      // what was loaded has been used, and every arrival of the matrix unit at this block's barriers is in:
      // the block may end
      for (int i = 0; i < kStages && i < loads; ++i) {
        if (stage-- == 0) stage = kStages - 1, phase ^= 1;
        if (ok) ok = dense_wait(empty + 8 * stage, phase);
        else if (rank == 0) dense_wait(full + 8 * stage, phase); // (copies in flight land before the way out)
      }
    }
  } else if (warp == 1) {
    if (lane == 0 && rank == 0) {
      int stage = 0, buf = 0;
      uint32_t phase = 0, tphase = 0;
      for (int unit = first; ok && unit < jobs.units; unit += step) of_job(unit, [&](const DenseProblem &p, const End &, int u) {
        const DenseUnit w = dense_unit(p, u);
        const uint32_t idesc = 1u << 4 | dense_format<T>() << 7 | dense_format<T>() << 10 | (uint32_t)p.a_rows_inner << 15 |
                               (uint32_t)p.b_rows_inner << 16 | (uint32_t)(BN / 8) << 17 | (uint32_t)((PAIR ? 256 : 128) / 16) << 24;
        const uint32_t a_step = p.a_rows_inner ? 2048 >> 4 : 32 >> 4, b_step = p.b_rows_inner ? 2048 >> 4 : 32 >> 4;
        // 64 k of a stage, rows block j, into accumulator `acc`
        auto multiply = [&](int at_stage, int j, int acc, bool fresh) {
          const uint32_t at = base + at_stage * kStageBytes;
          const uint64_t a = dense_desc(at + j * 16384, p.a_rows_inner), b = dense_desc(at + MT * 16384, p.b_rows_inner);
#pragma unroll
          for (int i = 0; i < kDenseK / 16; ++i)
            dense_mma<PAIR>(tmem + (uint32_t)(acc * BN), a + i * a_step, b + i * b_step, idesc, !fresh || i > 0);
        };
        for (int n = w.n0; ok && n < w.n1; ++n) {
          if constexpr (SHAPE == kDenseTall) {
            constexpr int kTail = 2;
            if (!(ok = dense_wait(tempty, tphase ^ 1))) break;
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            int behind = stage, lag = 0; // the second accumulator's next stage, and how many it is behind
            bool second = false, fresh = true;
            for (int k = w.k0; k < w.k1; ++k) {
              if (!(ok = dense_wait(full + 8 * stage, phase))) break;
              asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
              multiply(stage, 0, 0, k == w.k0);
              ++lag;
              if (++stage == kStages) stage = 0, phase ^= 1;
              const bool end = k == w.k1 - 1;
              if (end) dense_commit<PAIR>(tfull);
              if (!second) {
                if (lag == kStages || end) {
                  if (!(ok = dense_wait(tempty + 8, tphase ^ 1))) break;
                  second = true;
                } else {
                  second = dense_try(tempty + 8, tphase ^ 1);
                }
                if (second) asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
              }
              if (second && (end || k < w.k1 - kTail || lag == kStages))
                for (; lag > 0; --lag) {
                  multiply(behind, 1, 1, fresh);
                  fresh = false;
                  dense_commit<PAIR>(empty + 8 * behind);
                  if (++behind == kStages) behind = 0;
                }
            }
            if (!ok) break;
            dense_commit<PAIR>(tfull + 8);
            tphase ^= 1;
          } else {
            if (!(ok = dense_wait(tempty + 8 * buf, tphase ^ 1))) break;
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            for (int k = w.k0; k < w.k1; ++k) {
              if (!(ok = dense_wait(full + 8 * stage, phase))) break;
              asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
              multiply(stage, 0, buf, k == w.k0);
              dense_commit<PAIR>(empty + 8 * stage);
              if (++stage == kStages) stage = 0, phase ^= 1;
            }
            if (!ok) break;
            dense_commit<PAIR>(tfull + 8 * buf);
            if (++buf == 2) buf = 0, tphase ^= 1;
          }
        }
      });
    }
  } else if (warp >= 4) {
    const int e = warp - 4, part = e / 4;
    DenseWarp me{end_p + e * kDenseEndBytes, end_p + kDenseEndWarps * kDenseEndBytes + e * kDenseBiasBytes, own + 8 * e, 0, {0}, true, false};
    const uint32_t free_bar = PAIR ? dense_first(tempty) : tempty;
    int buf = 0;
    uint32_t tphase = 0;
    for (int unit = first; ok && unit < jobs.units; unit += step) of_job(unit, [&](const DenseProblem &p, const End &end, int u) {
      const DenseUnit w = dense_unit(p, u);
      const int row = w.m * BM + (int)rank * 128 + (warp % 4) * 32 + lane;
      typename End::State state[MT];
#pragma unroll
      for (int j = 0; j < MT; ++j) end.start(state[j], p, row + j * 256, w);
      for (int n = w.n0; ok && me.ok && n < w.n1; ++n) {
        const int col = n * BN + part * kColumns;
        end.tile(p, col, me);
#pragma unroll(sizeof(state) > 2 ? 2 : 1)
        for (int j = 0; j < MT; ++j) {
          if (MT == 2) buf = j;
          if (col < p.N) end.ahead(p, row + j * 256, col, kColumns, me);
          if (!(ok = __all_sync(~0u, dense_wait(tfull + 8 * buf, tphase)))) break;
          asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
          const uint32_t at = tmem + (uint32_t)(buf * BN + part * kColumns) + ((uint32_t)(warp % 4) << 21);
#pragma unroll 1
          for (int c = 0; c < kColumns; c += 32) {
            uint32_t r[32];
            __syncwarp();
            dense_take(at + c, r);
            dense_taken(r);
            if (c + 32 == kColumns) { // the accumulator is free as soon as its last values are in registers
              asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
              __syncwarp();
              if (lane == 0) {
                if constexpr (PAIR)
                  asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(free_bar + 8 * buf) : "memory");
                else
                  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(free_bar + 8 * buf) : "memory");
              }
            }
            if (col + c < p.N) end.chunk(state[j], p, r, row + j * 256, col + c, w, me, c > 0, c + 32 < kColumns && col + c + 32 < p.N);
          }
        }
        if (MT == 2) tphase ^= 1;
        else if (++buf == 2) buf = 0, tphase ^= 1;
      }
      ok = ok && me.ok;
      if (ok) {
#pragma unroll
        for (int j = 0; j < MT; ++j) end.stop(state[j], p, row + j * 256, w, part);
      }
    });
    if (lane == 0) {
      asm volatile("cp.async.bulk.wait_group 0;" ::: "memory"); // (stores under way read shared memory)
      if (me.coming) dense_wait(me.bar, me.phase);              // (after a wait that gave up: copies land before the way out)
    }
  }
  if (!ok) atomicExch(&tb_dense_status, 4);
  __syncwarp();
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  if constexpr (PAIR) {
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
  }
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  if (warp == 2) {
    if constexpr (PAIR) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(2 * BN) : "memory");
    else asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(2 * BN) : "memory");
  }
}

// ---- what becomes of a tile ---------------------------------------------------------------------

__device__ __forceinline__ float exp2_fast(float x) { // within 2 steps of 2^-23; below 2^-126: 0
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float inverse_fast(float x) { // within a step of 2^-23
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
constexpr float kLog2e = 1.44269504f;

// Two fp32 operations in one instruction.
struct Two {
  unsigned long long v;
  __device__ __forceinline__ Two() {}
  __device__ __forceinline__ Two(float a, float b) { asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(a), "f"(b)); }
  __device__ __forceinline__ explicit Two(float a) : Two(a, a) {}
  __device__ __forceinline__ explicit Two(float2 a) : Two(a.x, a.y) {}
  __device__ __forceinline__ float2 get() const {
    float2 f;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(f.x), "=f"(f.y) : "l"(v));
    return f;
  }
};
__device__ __forceinline__ Two operator+(Two a, Two b) {
  Two r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
__device__ __forceinline__ Two operator*(Two a, Two b) {
  Two r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
__device__ __forceinline__ Two fma2(Two a, Two b, Two c) {
  Two r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v));
  return r;
}

// -Phi(-|z|), Phi the integral of the normal distribution, and exp(-z^2 / 2), of two z.  erfc's shape after Hastings
// (Approximations for Digital Computers, 1955): Phi(-|z|) = exp(-z^2 / 2) t P(t), t = 1 / (1 + 0.33 |z|);
// P was fitted here, by reweighted least squares, for the relative error, 1e-6.  In fp32, with the exponential of a
// rounded square, it is 2e-6 + z^2 2^-24 up to |z| = 13, beyond which the exponential is 0; |z| times it, what gelu takes
// off max(z, 0), is off by less than 4e-7.  Without branches, since a warp's values need both sides of any (the
// library's erff took most of a layer's time).
__device__ __forceinline__ Two normal_tail(float2 z, float2 size, float2 *bell) { // size: |z|, finite
  const Two zz(z), a(size);
  const float2 d = fma2(a, Two(0.33f), Two(1.f)).get();
  const Two t(inverse_fast(d.x), inverse_fast(d.y));
  Two p = fma2(Two(-0.0332859295f), t, Two(0.105665717f));
  p = fma2(p, t, Two(-0.067432403f));
  p = fma2(p, t, Two(-0.0334278586f));
  p = fma2(p, t, Two(-0.0910052722f));
  p = fma2(p, t, Two(-0.117216671f));
  p = fma2(p, t, Two(-0.13164699f));
  p = fma2(p, t, Two(-0.131651081f));
  const float2 e = (zz * (zz * Two(-0.5f * kLog2e))).get();
  *bell = make_float2(exp2_fast(e.x), exp2_fast(e.y));
  return Two(*bell) * (t * p);
}
__device__ __forceinline__ float2 size_of(float2 z) { // (an infinite z has tail 0)
  return make_float2(fminf(fabsf(z.x), 1e18f), fminf(fabsf(z.y), 1e18f));
}
enum { kActNone = 0, kActRelu = 1, kActGelu = 2, kActSilu = 3 };
template <int ACT> __device__ __forceinline__ float2 act_value(float2 z) {
  if constexpr (ACT == kActRelu) return make_float2(z.x < 0.f ? 0.f : z.x, z.y < 0.f ? 0.f : z.y); // (NaN stays)
  if constexpr (ACT == kActGelu) { // z Phi(z) = max(z, 0) - |z| Phi(-|z|)
    float2 bell;
    const float2 a = size_of(z);
    return fma2(Two(a), normal_tail(z, a, &bell), Two(fmaxf(z.x, 0.f), fmaxf(z.y, 0.f))).get();
  }
  if constexpr (ACT == kActSilu)
    return make_float2(z.x * inverse_fast(1.f + exp2_fast(-kLog2e * z.x)), z.y * inverse_fast(1.f + exp2_fast(-kLog2e * z.y)));
  return z;
}
// An infinite z, as the rounding of a kept value to fp16 can bring, has the slope of a large one: without this it
// would be infinity times the 0 of the tail.
__device__ __forceinline__ float finite(float z) { return fabsf(z) == INFINITY ? copysignf(1e30f, z) : z; }
template <int ACT> __device__ __forceinline__ float2 act_slope(float2 z) {
  if constexpr (ACT == kActGelu || ACT == kActSilu) z = make_float2(finite(z.x), finite(z.y));
  if constexpr (ACT == kActRelu) return make_float2(z.x > 0.f ? 1.f : 0.f, z.y > 0.f ? 1.f : 0.f);
  if constexpr (ACT == kActGelu) { // Phi(z) + z phi(z)
    float2 bell;
    const float2 tail = normal_tail(z, size_of(z), &bell).get();
    return make_float2(fmaf(z.x * 0.39894228f, bell.x, z.x >= 0.f ? 1.f + tail.x : -tail.x), fmaf(z.y * 0.39894228f, bell.y, z.y >= 0.f ? 1.f + tail.y : -tail.y));
  }
  if constexpr (ACT == kActSilu) {
    const float s = inverse_fast(1.f + exp2_fast(-kLog2e * z.x)), t = inverse_fast(1.f + exp2_fast(-kLog2e * z.y));
    return make_float2(s * fmaf(z.x, 1.f - s, 1.f), t * fmaf(z.y, 1.f - t, 1.f));
  }
  return make_float2(1.f, 1.f);
}
// f(activation as a constant): one test for all of a thread's values
template <class F> __device__ __forceinline__ void with_act(int act, F f) {
  switch (act) {
  case kActRelu: f(std::integral_constant<int, kActRelu>()); break;
  case kActGelu: f(std::integral_constant<int, kActGelu>()); break;
  case kActSilu: f(std::integral_constant<int, kActSilu>()); break;
  }
}

template <class T> __device__ __forceinline__ uint32_t pack2(float a, float b);
template <> __device__ __forceinline__ uint32_t pack2<__half>(float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t *>(&h);
}
template <> __device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float a, float b) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t *>(&h);
}
template <class T> __device__ __forceinline__ float2 unpack2(uint32_t w) {
  if constexpr (std::is_same<T, __half>::value) return __half22float2(*reinterpret_cast<const __half2 *>(&w));
  else return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}
// Eight consecutive elements, `n` of them there; `vec`: 16-byte aligned.
template <class T> __device__ __forceinline__ void store8(T *p, const float (&v)[8], int n, bool vec) {
  if (vec && n >= 8) {
    *reinterpret_cast<uint4 *>(p) = make_uint4(pack2<T>(v[0], v[1]), pack2<T>(v[2], v[3]), pack2<T>(v[4], v[5]), pack2<T>(v[6], v[7]));
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < n) p[i] = from_float<T>(v[i]);
  }
}
template <class T> __device__ __forceinline__ void load8(const T *p, float (&v)[8], int n, bool vec) {
  if (vec && n >= 8) {
    const uint4 q = *reinterpret_cast<const uint4 *>(p);
    const T *h = reinterpret_cast<const T *>(&q);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = to_float(h[i]);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = i < n ? to_float(p[i]) : 0.f;
  }
}

template <class T> __device__ __forceinline__ uint4 raw8(const T *p, int n, bool vec) { // eight elements as they are, n of them there
  if (vec && n >= 8) return *reinterpret_cast<const uint4 *>(p);
  uint32_t w[4] = {0, 0, 0, 0};
  const unsigned short *q = reinterpret_cast<const unsigned short *>(p);
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if (i < n) w[i / 2] |= (uint32_t)q[i] << (i % 2 * 16);
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// Results on their way out: a warp puts 32 rows x 32 columns (a row is 64 bytes, its 16-byte pieces swapped
// around by the row's number, as the tensor map says) into its shared memory and one tensor copy takes them to
// where they belong; what is behind the last row or column the copy leaves out.
constexpr int kOutBytes = 2048;
template <int BUT> __device__ __forceinline__ void out_free() { // all copies but the last BUT have read the shared memory
  if (threadIdx.x % 32 == 0) asm volatile("cp.async.bulk.wait_group.read %0;" ::"n"(BUT) : "memory");
  __syncwarp();
}
// The same before `pieces` of the warp's shared memory are written and copied out.
__device__ __forceinline__ void out_claim(DenseWarp &w, uint32_t pieces) {
  if (w.out.claim(pieces)) out_free<1>();
  else out_free<0>();
}
__device__ __forceinline__ uint4 *out_piece(unsigned char *buf, int i) { // the lane's row's columns 8 i ...
  const int lane = threadIdx.x % 32;
  return reinterpret_cast<uint4 *>(buf) + lane * 4 + (i ^ (lane >> 1 & 3));
}
template <class T> __device__ __forceinline__ void out_put(unsigned char *buf, const Two (&v)[16]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 a = v[4 * i].get(), b = v[4 * i + 1].get(), c = v[4 * i + 2].get(), d = v[4 * i + 3].get();
    *out_piece(buf, i) = make_uint4(pack2<T>(a.x, a.y), pack2<T>(b.x, b.y), pack2<T>(c.x, c.y), pack2<T>(d.x, d.y));
  }
}
__device__ __forceinline__ void out_ready() { // (of all lanes, before one of them sends)
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  __syncwarp();
}
__device__ __forceinline__ void out_send(const CUtensorMap *map, const unsigned char *buf, int m, int n) {
  asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.tile.bulk_group [%0, {%1, %2}], [%3];"
               ::"l"(map), "r"(n), "r"(m), "r"(dense_smem(buf)) : "memory");
}
__device__ __forceinline__ void out_send3(const CUtensorMap *map, const unsigned char *buf, int split, int m, int n) {
  asm volatile("cp.async.bulk.tensor.3d.global.shared::cta.tile.bulk_group [%0, {%1, %2, %3}], [%4];"
               ::"l"(map), "r"(n), "r"(m), "r"(split), "r"(dense_smem(buf)) : "memory");
}
__device__ __forceinline__ void out_commit() { asm volatile("cp.async.bulk.commit_group;" ::: "memory"); }

// 32 rows x 32 fp32 values turned around in shared memory, 16-byte pieces swapped around by the row's number,
// which keeps both directions free of bank conflicts.  f(row, column 0, 8, 16 or 24, eight values).
__device__ __forceinline__ void turn(const uint32_t (&r)[32], unsigned char *mine) {
  const int lane = threadIdx.x % 32;
  uint4 *s = reinterpret_cast<uint4 *>(mine);
  __syncwarp();
#pragma unroll
  for (int i = 0; i < 8; ++i) s[lane * 8 + (i ^ (lane & 7))] = make_uint4(r[4 * i], r[4 * i + 1], r[4 * i + 2], r[4 * i + 3]);
  __syncwarp();
}
template <class F> __device__ __forceinline__ void turned(const unsigned char *mine, F f) {
  const int lane = threadIdx.x % 32;
  const float4 *s = reinterpret_cast<const float4 *>(mine);
#pragma unroll 1
  for (int i = 0; i < 4; ++i) {
    const int row = i * 8 + lane / 4, c = lane % 4;
    const float4 x = s[row * 8 + ((2 * c) ^ (row & 7))], y = s[row * 8 + ((2 * c + 1) ^ (row & 7))];
    const float w[8] = {x.x, x.y, x.z, x.w, y.x, y.y, y.z, y.w};
    f(row, c * 8, w);
  }
}

// The same pieces of 32 rows x 32 columns to and from matrices whose rows begin anywhere, which tensor copies cannot
// reach: a lane per column, 32 neighbouring elements at a time.  (Calls, as everything that few products need, so
// that the way of the others stays short: their instructions come from a small cache.)
template <class T> __device__ __forceinline__ T *out_element(unsigned char *buf, int row) {
  const int lane = threadIdx.x % 32;
  return reinterpret_cast<T *>(buf) + row * 32 + (((lane >> 3) ^ (row >> 1 & 3)) << 3 | (lane & 7));
}
template <class T> __device__ __noinline__ void copy_out(T *to, long long ld, int m0, int n, int M, int N, unsigned char *buf) {
  __syncwarp();
  if (n + (int)(threadIdx.x % 32) < N) {
    T *p = to + (long long)m0 * ld + n + threadIdx.x % 32;
    const int rows = min(32, M - m0);
#pragma unroll 8
    for (int r = 0; r < rows; ++r) p[r * ld] = *out_element<T>(buf, r);
  }
  __syncwarp();
}
template <class T> __device__ __noinline__ void copy_in(const T *from, long long ld, int m0, int n, int M, int N, unsigned char *buf) {
  __syncwarp();
  const bool there = n + (int)(threadIdx.x % 32) < N;
  const T *p = from + (long long)m0 * ld + n + threadIdx.x % 32;
#pragma unroll 8
  for (int r = 0; r < 32; ++r) *out_element<T>(buf, r) = there && m0 + r < M ? p[r * ld] : from_float<T>(0.f);
  __syncwarp();
}

// What a whole sum c becomes: z = c / scale + bias; out = activation(z) + addend; pre = z.  Or, with `sums`, one
// piece of a longer sum, added to the pieces before it.  With `parts` the sum is cut into parts, which are kept:
// parts[split][row][ld_parts].
template <class T> struct Result {
  CUtensorMap parts_map; // of `parts`
  CUtensorMap out_map, pre_map, addend_map; // where the matrix's rows lie at multiples of 16 bytes (tma_*)
  const T *bias, *addend;
  T *out, *pre;
  float *sums; // [rows][ld_sums] or null
  float *parts; // or null
  const float *scale; // a power of two, or null
  long long ld_addend, ld_out, ld_pre, ld_sums, ld_parts;
  int act;
  bool first, last;                                   // piece of a sum
  bool tma_addend, tma_out, tma_pre;                  // tensor copies reach the matrix
  bool vec_addend, vec_out, vec_pre, vec_bias;        // every eighth column lies at a multiple of 16 bytes
  __device__ __forceinline__ void finish8(const float (&c)[8], long long m, long long n, long long N) const {
    const int have = (int)min(8ll, N - n);
    float z[8], b[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) z[i] = c[i];
    if (sums) {
      float4 *s = reinterpret_cast<float4 *>(sums + m * ld_sums + n); // (ld a multiple of 8: whole pieces of 8 are there)
      if (!first) {
        const float4 x = s[0], y = s[1];
        z[0] += x.x, z[1] += x.y, z[2] += x.z, z[3] += x.w, z[4] += y.x, z[5] += y.y, z[6] += y.z, z[7] += y.w;
      }
      if (!last) {
        s[0] = make_float4(z[0], z[1], z[2], z[3]);
        s[1] = make_float4(z[4], z[5], z[6], z[7]);
        return;
      }
    }
    if (scale) {
      const float d = 1.f / *scale;
#pragma unroll
      for (int i = 0; i < 8; ++i) z[i] *= d;
    }
    if (bias) {
      load8(bias + n, b, have, vec_bias);
#pragma unroll
      for (int i = 0; i < 8; ++i) z[i] += b[i];
    }
    if (pre) store8(pre + m * ld_pre + n, z, have, vec_pre);
    with_act(act, [&](auto a) {
#pragma unroll
      for (int i = 0; i < 8; i += 2) {
        const float2 y = act_value<decltype(a)::value>(make_float2(z[i], z[i + 1]));
        z[i] = y.x, z[i + 1] = y.y;
      }
    });
    if (addend) {
      load8(addend + m * ld_addend + n, b, have, vec_addend);
#pragma unroll
      for (int i = 0; i < 8; ++i) z[i] += b[i];
    }
    store8(out + m * ld_out + n, z, have, vec_out);
  }
};

// A warp's 32 x 32 sums, turned around in its shared memory, to where pieces of sums are kept.
template <class T> __device__ __noinline__ void keep_sums(const Result<T> &f, const unsigned char *mine, int m0, int n, int M, int N) {
  turned(mine, [&](int k, int c, const float (&x)[8]) {
    if (m0 + k < M && n + c < N) f.finish8(x, m0 + k, n + c, N);
  });
}

// Finishes sums, a row per lane.  Addends come, and results go, 32 rows x 32 columns at a time through shared memory,
// by tensor copies where these reach the matrix.  (Reading them a row per lane took longer than the product.)  A warp
// has two pieces of 2 KB, which results go through by turns; addends that tensor copies bring come there, one for
// each half of the warp's columns, before the sums are done, and the results replace them; where z is kept too, the
// second is z's, and parts of sums take both.  The two products of a launch use them differently: see OutPieces.
template <class T> struct ResultEnd {
  Result<T> f;
  struct State {};
  __device__ __forceinline__ void start(State &, const DenseProblem &, int, const DenseUnit &) const {}
  __device__ __forceinline__ void tile(const DenseProblem &p, int n, DenseWarp &w) const {
    if (!f.bias) return;
    T *b = reinterpret_cast<T *>(w.bias);
    __syncwarp();
#pragma unroll
    for (int i = threadIdx.x % 32; i < 64; i += 32) { // (of the 64 columns that the warp's lie in)
      const int c = n - n % 64 + i;
      b[i] = c < p.N ? f.bias[c] : from_float<T>(0.f);
    }
    __syncwarp();
  }
  __device__ __forceinline__ void fetch(int row, int n, unsigned char *to, DenseWarp &w) const {
    dense_load<false>(dense_smem(to), &f.addend_map, n, row, w.bar);
  }
  // (row: the lane's; the first lane's is the warp's first)
  __device__ __forceinline__ void ahead(const DenseProblem &p, int row, int n, int columns, DenseWarp &w) const {
    if (!f.addend || !f.tma_addend || f.parts || !w.ok || threadIdx.x % 32) return;
    const bool two = columns > 32 && n + 32 < p.N && !f.pre;
    asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory"); // (the last results may still be on their way)
    dense_expect(w.bar, two ? 2 * kOutBytes : kOutBytes);
    w.coming = true;
    fetch(row, n, w.mine, w);
    if (two) fetch(row, n + 32, w.mine + kOutBytes, w);
  }
  __device__ __forceinline__ void chunk(State &, const DenseProblem &p, const uint32_t (&r)[32], int row, int n, const DenseUnit &u,
                                        DenseWarp &w, bool second, bool more) const {
    const int lane = threadIdx.x % 32;
    const int m0 = row - lane;
    if (f.parts) { // (4 KB a time, turned around as their map says)
      out_claim(w, 3);
      turn(r, w.mine);
      out_ready();
      if (lane == 0) {
        if (m0 < p.M) out_send3(&f.parts_map, w.mine, u.split, m0, n);
        out_commit();
      }
      return;
    }
    if (f.sums) {
      out_claim(w, 3);
      w.out.read = 0; // (nothing is copied out of it)
      turn(r, w.mine);
      return keep_sums(f, w.mine, m0, n, p.M, p.N);
    }
    Two z[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) z[i] = Two(__uint_as_float(r[2 * i]), __uint_as_float(r[2 * i + 1]));
    if (f.scale) {
      const Two d(1.f / *f.scale);
#pragma unroll
      for (int i = 0; i < 16; ++i) z[i] = z[i] * d;
    }
    auto add8 = [&](int i, uint4 q) {
      add_halves<T>(z[4 * i].v, q.x);
      add_halves<T>(z[4 * i + 1].v, q.y);
      add_halves<T>(z[4 * i + 2].v, q.z);
      add_halves<T>(z[4 * i + 3].v, q.w);
    };
    if (f.bias) {
      const uint4 *b = reinterpret_cast<const uint4 *>(w.bias) + n % 64 / 8;
#pragma unroll
      for (int i = 0; i < 4; ++i) add8(i, b[i]);
    }
    const uint32_t pieces = f.pre ? 3 : f.addend ? (second ? 2 : 1) : w.out.other();
    unsigned char *to = w.mine + (pieces == 2 ? kOutBytes : 0), *kept = w.mine + kOutBytes;
    out_claim(w, pieces);
    if (f.addend) {
      if (!f.tma_addend) {
        copy_in(f.addend, f.ld_addend, m0, n, p.M, p.N, to);
      } else if (!second || f.pre) {
        if (w.ok && (w.ok = __all_sync(~0u, dense_wait(w.bar, w.phase)))) w.phase ^= 1, w.coming = false;
      }
    }
    if (f.pre) out_put<T>(kept, z);
    with_act(f.act, [&](auto a) {
#pragma unroll
      for (int i = 0; i < 16; ++i) z[i] = Two(act_value<decltype(a)::value>(z[i].get()));
    });
    if (f.addend) {
#pragma unroll
      for (int i = 0; i < 4; ++i) add8(i, *out_piece(to, i));
    }
    out_put<T>(to, z);
    if (f.pre && !f.tma_pre) copy_out(f.pre, f.ld_pre, m0, n, p.M, p.N, kept);
    if (!f.tma_out) copy_out(f.out, f.ld_out, m0, n, p.M, p.N, to);
    out_ready();
    if (lane == 0) {
      if (m0 < p.M) {
        if (f.tma_out) out_send(&f.out_map, to, m0, n);
        if (f.pre && f.tma_pre) out_send(&f.pre_map, kept, m0, n);
      }
      out_commit();
      if (more && f.addend && f.tma_addend && f.pre && w.ok) { // (no room for it before)
        asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
        dense_expect(w.bar, kOutBytes);
        w.coming = true;
        fetch(m0, n + 32, w.mine, w);
      }
    }
  }
  __device__ __forceinline__ void stop(State &, const DenseProblem &, int, const DenseUnit &, int) const {}
};
// Adds parts up, in order, and finishes them; adds up rows of column sums.  One launch for what follows a call's
// products: blocks 0 .. blocks[0] - 1 have the first job, and so on.
template <class T> struct FinishJobs {
  unsigned blocks[3];
  int splits[2];
  long long M[2], N[2];
  Result<T> end[2]; // end.parts, end.ld_parts
  const float *rows; // [count][ld_rows]
  long long count, ld_rows, columns;
  T *column_sums;     // sum of a column of `rows` / *scale
  const float *scale; // or null: 1
};
template <class T>
__device__ __forceinline__ void join_parts(const Result<T> &f, int splits, long long M, long long N, unsigned block) {
  const long long per = f.ld_parts / 8, i = (long long)block * 256 + threadIdx.x;
  if (i >= M * per) return;
  const long long m = i / per, n = i % per * 8;
  float v[8] = {};
#pragma unroll 4
  for (int s = 0; s < splits; ++s) {
    const float4 *d = reinterpret_cast<const float4 *>(f.parts + ((long long)s * M + m) * f.ld_parts + n);
    const float4 a = d[0], b = d[1];
    v[0] += a.x, v[1] += a.y, v[2] += a.z, v[3] += a.w, v[4] += b.x, v[5] += b.y, v[6] += b.z, v[7] += b.w;
  }
  f.finish8(v, m, n, N);
}
template <class T> __global__ void __launch_bounds__(256) tb_dense_finish_kernel(const __grid_constant__ FinishJobs<T> jobs) {
  __shared__ float part[8][32];
  after_previous_kernel();
  unsigned b = blockIdx.x;
  if (b < jobs.blocks[0]) return join_parts(jobs.end[0], jobs.splits[0], jobs.M[0], jobs.N[0], b);
  b -= jobs.blocks[0];
  if (b < jobs.blocks[1]) return join_parts(jobs.end[1], jobs.splits[1], jobs.M[1], jobs.N[1], b);
  b -= jobs.blocks[1];
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  const long long c = (long long)b * 32 + lane;
  float s = 0.f;
  if (c < jobs.columns)
#pragma unroll 8
    for (long long t = warp; t < jobs.count; t += 8) s += jobs.rows[t * jobs.ld_rows + c];
  part[warp][lane] = s;
  __syncthreads();
  if (warp || c >= jobs.columns) return;
#pragma unroll
  for (int i = 1; i < 8; ++i) s += part[i][lane];
  jobs.column_sums[c] = from_float<T>(jobs.scale ? s / *jobs.scale : s);
}

// ---- few rows ---------------------------------------------------------------------------------------
// y for up to ROWS rows of x: a warp per output reads its row of the weights once, eight elements a lane at a time
// (in one read where VEC), four of these under way; what bounds it is the latency of one such read, then the
// weights' bytes.
constexpr int kFewRows = 8;
template <class T, bool VEC, int ROWS>
__global__ void __launch_bounds__(256) tb_linear_rows_kernel(const T *x, long long ld_x, const T *weight, long long ld_w,
                                                             const __grid_constant__ Result<T> f, int rows, int inputs, int outputs) {
  constexpr int kPer = 8, kAhead = 4;
  after_previous_kernel();
  const int lane = threadIdx.x % 32;
  auto read = [&](const T *p, int k) { return k < inputs ? raw8(p + k, min(8, inputs - k), VEC) : make_uint4(0, 0, 0, 0); };
  for (long long o = (long long)blockIdx.x * 8 + threadIdx.x / 32; o < outputs; o += gridDim.x * 8ll) {
    Two acc[ROWS];
#pragma unroll
    for (int r = 0; r < ROWS; ++r) acc[r] = Two(0.f);
    const T *row = weight + o * ld_w;
    for (int k0 = lane * kPer; k0 < inputs; k0 += 32 * kPer * kAhead) {
      uint4 w[kAhead];
#pragma unroll
      for (int i = 0; i < kAhead; ++i) w[i] = read(row, k0 + i * 32 * kPer);
#pragma unroll
      for (int i = 0; i < kAhead; ++i) {
        const uint32_t ww[4] = {w[i].x, w[i].y, w[i].z, w[i].w};
#pragma unroll
        for (int r = 0; r < ROWS; ++r) {
          const uint4 q = read(x + (r < rows ? r : 0) * ld_x, k0 + i * 32 * kPer);
          const uint32_t qw[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
          for (int j = 0; j < 4; ++j) acc[r] = fma2(Two(unpack2<T>(ww[j])), Two(unpack2<T>(qw[j])), acc[r]);
        }
      }
    }
    float sum[ROWS];
#pragma unroll
    for (int r = 0; r < ROWS; ++r) {
      const float2 v = acc[r].get();
      sum[r] = v.x + v.y;
#pragma unroll
      for (int d = 16; d; d >>= 1) sum[r] += __shfl_xor_sync(~0u, sum[r], d);
    }
    float mine = 0.f;
#pragma unroll
    for (int r = 0; r < ROWS; ++r)
      if (lane == r) mine = sum[r];
    if (lane < rows) {
      const float z = f.bias ? mine + to_float(f.bias[o]) : mine;
      if (f.pre) f.pre[lane * f.ld_pre + o] = from_float<T>(z);
      float y = z;
      with_act(f.act, [&](auto a) { y = act_value<decltype(a)::value>(make_float2(z, z)).x; });
      f.out[lane * f.ld_out + o] = from_float<T>(f.addend ? y + to_float(f.addend[lane * f.ld_addend + o]) : y);
    }
  }
}

__device__ __forceinline__ long long label_at(const void *labels, int bytes, long long m) {
  return bytes == 8 ? static_cast<const long long *>(labels)[m] : static_cast<const int *>(labels)[m];
}
// The biases of a warp's 64 (or 32) columns of a tile, in its shared memory; -inf for columns behind the last class,
// which thereby have probability 0.
template <class T, int COLS>
__device__ __forceinline__ void stage_bias(const T *bias, int n, int N, float *dst) {
  __syncwarp();
#pragma unroll
  for (int i = threadIdx.x % 32; i < COLS; i += 32) dst[i] = n + i >= N ? -INFINITY : bias ? to_float(bias[n + i]) : 0.f;
  __syncwarp();
}

__device__ __forceinline__ float max3(float a, float b, float c) { // (not a number: the others)
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}

// What is subtracted from scores whose largest is `top`: nothing where that is infinite (all so far forbidden, their
// exponentials are 0; or infinite, and the sum with it).
__device__ __forceinline__ float lse_ref(float top) { return fabsf(top) == INFINITY ? 0.f : top; }

// Sum of a row's exponentials over the tiles of a unit, relative to the largest score of them, in one pass:
// the sum so far is scaled down whenever a larger score comes.  Scores become powers of two after the largest has
// been subtracted (an operation more for two scores than scaling them first; 4096 x 100003 scores: 64 columns 151 to
// 158 us, 256 columns 187 to 193, 512 columns 330 to 335): so that the largest one's exponential is 1, sums are 1 or more
// and no loss falls below 0.  parts[4 * chunk + part][row]
template <class T, int COLS> struct LseEnd {
  const T *bias;
  const void *labels;
  int label_bytes;
  float2 *parts;
  float *at; // [rows] the label's score
  struct State {
    float top, sum;
    int label;
  };
  __device__ __forceinline__ void start(State &s, const DenseProblem &p, int row, const DenseUnit &) const {
    s.top = -INFINITY;
    s.sum = 0.f;
    const long long label = row < p.M ? label_at(labels, label_bytes, row) : -1;
    s.label = label >= 0 && label < p.N ? (int)label : -1;
  }
  __device__ __forceinline__ void tile(const DenseProblem &p, int n, DenseWarp &w) const {
    stage_bias<T, COLS>(bias, n, p.N, reinterpret_cast<float *>(w.bias));
  }
  __device__ __forceinline__ void ahead(const DenseProblem &, int, int, int, DenseWarp &) const {}
  __device__ __forceinline__ void chunk(State &s, const DenseProblem &p, const uint32_t (&r)[32], int row, int n, const DenseUnit &,
                                        DenseWarp &w, bool, bool) const {
    const int at_label = s.label - n;
    if (s.label >= 0 && at_label >= 0 && at_label < 32) { // (the score itself, not its multiple)
      float z = 0.f;
#pragma unroll
      for (int j = 0; j < 32; ++j)
        if (j == at_label) z = __uint_as_float(r[j]);
      at[row] = bias ? z + to_float(bias[s.label]) : z;
    }
    const ulonglong2 *b2 = reinterpret_cast<const ulonglong2 *>(w.bias) + n % COLS / 4;
    Two z[16];
    float tops[2] = {s.top, s.top};
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const ulonglong2 b = b2[j];
      Two lo, hi;
      lo.v = b.x, hi.v = b.y;
      z[2 * j] = Two(__uint_as_float(r[4 * j]), __uint_as_float(r[4 * j + 1])) + lo;
      z[2 * j + 1] = Two(__uint_as_float(r[4 * j + 2]), __uint_as_float(r[4 * j + 3])) + hi;
      const float2 x = z[2 * j].get(), y = z[2 * j + 1].get();
      tops[j & 1] = max3(tops[j & 1], x.x, x.y);
      tops[j & 1] = max3(tops[j & 1], y.x, y.y);
    }
    const float top = fmaxf(tops[0], tops[1]), ref = lse_ref(top);
    const Two less(-ref);
    Two sum[2] = {Two(0.f), Two(0.f)};
#pragma unroll
    for (int j = 0; j < 16; ++j) {
      const float2 x = ((z[j] + less) * Two(kLog2e)).get();
      sum[j & 1] = sum[j & 1] + Two(exp2_fast(x.x), exp2_fast(x.y));
    }
    const float2 x = (sum[0] + sum[1]).get();
    s.sum = s.sum * exp2_fast((s.top - ref) * kLog2e) + (x.x + x.y);
    s.top = top;
  }
  __device__ __forceinline__ void stop(State &s, const DenseProblem &p, int row, const DenseUnit &u, int part) const {
    if (row < p.M) parts[(4ll * u.chunk + part) * p.M + row] = make_float2(s.top, s.sum);
  }
};

// A row's logarithm and loss from its parts: a lane per row, the parts over the block's warps (kJoinWarps at most).
constexpr int kJoinWarps = 32;
__global__ void __launch_bounds__(32 * kJoinWarps) tb_loss_join_kernel(const float2 *parts, int count, const float *at, const void *labels, int label_bytes,
                                                                       long long classes, float *loss, float *lse, long long rows) {
  __shared__ float2 mine[kJoinWarps][32];
  after_previous_kernel();
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32, warps = blockDim.x / 32;
  const long long m = (long long)blockIdx.x * 32 + lane;
  float top = -INFINITY, sum = 0.f;
  auto join = [&](float2 q) {
    const float most = fmaxf(top, q.x), ref = lse_ref(most);
    sum = sum * exp2_fast((top - ref) * kLog2e) + q.y * exp2_fast((q.x - ref) * kLog2e);
    top = most;
  };
  if (m < rows) {
#pragma unroll 4
    for (int t = warp; t < count; t += warps) join(parts[(long long)t * rows + m]);
  }
  mine[warp][lane] = make_float2(top, sum);
  __syncthreads();
  if (warp || m >= rows) return;
#pragma unroll 4
  for (int w = 1; w < warps; ++w) join(mine[w][lane]);
  const float most = top == -INFINITY ? 0.f : top, rest = logf(sum);
  const long long label = label_at(labels, label_bytes, m);
  lse[m] = most + rest;
  loss[m] = label >= 0 && label < classes ? (most - at[m]) + rest : 0.f; // (the label's score is subtracted before digits are lost)
}

// dz = weight * (exp(z - lse) - [label]) * scale, rounded, and the sums of its columns over 32 rows before
// that: bias_sums[row / 32][ld]
template <class T, int COLS> struct ScoreGradEnd {
  CUtensorMap dz_map;
  const T *bias; // of the piece's first class
  const void *labels;
  int label_bytes;
  const float *grad, *lse, *scale;
  long long ld, first, classes; // of bias_sums; class of column 0, all classes
  float *bias_sums;
  struct State {
    float weight, lse;
    int label; // column, or behind the last one
  };
  __device__ __forceinline__ void start(State &s, const DenseProblem &p, int row, const DenseUnit &) const {
    s.weight = s.lse = 0.f;
    s.label = 0x7fffffff;
    if (row >= p.M) return;
    const long long label = label_at(labels, label_bytes, row);
    if (label < 0 || label >= classes) return; // (its dz are zeros whatever the scores)
    if (label >= first && label < first + p.N) s.label = (int)(label - first);
    s.weight = grad[row] * *scale;
    s.lse = lse[row];
  }
  __device__ __forceinline__ void tile(const DenseProblem &p, int n, DenseWarp &w) const {
    stage_bias<T, COLS>(bias, n, p.N, reinterpret_cast<float *>(w.bias));
  }
  __device__ __forceinline__ void ahead(const DenseProblem &, int, int, int, DenseWarp &) const {}
  __device__ __forceinline__ void chunk(State &s, const DenseProblem &p, const uint32_t (&r)[32], int row, int n, const DenseUnit &,
                                        DenseWarp &w, bool, bool) const {
    const int lane = threadIdx.x % 32;
    const uint32_t piece = w.out.other();
    unsigned char *mine = w.mine + (piece == 2 ? kOutBytes : 0);
    const ulonglong2 *b2 = reinterpret_cast<const ulonglong2 *>(w.bias) + n % COLS / 4;
    const Two less(-s.lse), weight(s.weight);
    Two v[16];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const ulonglong2 b = b2[j];
      Two lo, hi;
      lo.v = b.x, hi.v = b.y;
      const float2 x = ((Two(__uint_as_float(r[4 * j]), __uint_as_float(r[4 * j + 1])) + lo + less) * Two(kLog2e)).get();
      const float2 y = ((Two(__uint_as_float(r[4 * j + 2]), __uint_as_float(r[4 * j + 3])) + hi + less) * Two(kLog2e)).get();
      v[2 * j] = Two(exp2_fast(x.x), exp2_fast(x.y)) * weight;
      v[2 * j + 1] = Two(exp2_fast(y.x), exp2_fast(y.y)) * weight;
    }
    if (s.weight == 0.f) { // (a score may be infinite)
#pragma unroll
      for (int j = 0; j < 16; ++j) v[j] = Two(0.f);
    }
    const int at = s.label - n;
    if (at >= 0 && at < 32) {
#pragma unroll
      for (int j = 0; j < 16; ++j) {
        const float2 x = v[j].get();
        v[j] = Two(2 * j == at ? x.x - s.weight : x.x, 2 * j + 1 == at ? x.y - s.weight : x.y);
      }
    }
    out_claim(w, piece);
    out_put<T>(mine, v);
    const int m0 = row - lane;
    out_ready();
    if (lane == 0) {
      if (m0 < p.M) out_send(&dz_map, mine, m0, n);
      out_commit();
    }
    if (bias_sums) {
      // sums over the 32 lanes of 32 values each: every step halves the values and doubles the lanes summed
      float c[32];
#pragma unroll
      for (int j = 0; j < 16; ++j) {
        const float2 x = v[j].get();
        c[2 * j] = x.x, c[2 * j + 1] = x.y;
      }
#pragma unroll
      for (int d = 16; d; d >>= 1) {
        const bool upper = lane & d;
#pragma unroll
        for (int j = 0; j < d; ++j) {
          const float keep = upper ? c[j + d] : c[j], give = upper ? c[j] : c[j + d];
          c[j] = keep + __shfl_xor_sync(~0u, give, d);
        }
      }
      if (m0 < p.M && n + lane < ld) bias_sums[(long long)(m0 / 32) * ld + n + lane] = c[0];
    }
  }
  __device__ __forceinline__ void stop(State &, const DenseProblem &, int, const DenseUnit &, int) const {}
};

// dz = grad * activation'(pre), rounded; sums of its columns over 32 rows before that.  32 rows x 256 columns
// a block, four rows a warp, whose loads are under way together.
template <class T, int ACT>
__device__ __forceinline__ void act_grad(const T *grad, long long ld_grad, bool vec_grad, const T *pre, long long ld_pre, bool vec_pre, T *dz,
                                         long long ld, float *bias_sums, int rows, int cols, int bx, int by, float (&part)[8][256]) {
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  const int c = (by * 32 + lane) * 8, r0 = bx * 32 + warp * 4, have = min(8, cols - c);
  float sum[8] = {};
  if (have > 0) {
    uint4 g[4], z[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) g[i] = raw8(grad + (r0 + i) * ld_grad + c, r0 + i < rows ? have : 0, vec_grad);
    if constexpr (ACT != kActNone) {
#pragma unroll
      for (int i = 0; i < 4; ++i) z[i] = raw8(pre + (r0 + i) * ld_pre + c, r0 + i < rows ? have : 0, vec_pre);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t gw[4] = {g[i].x, g[i].y, g[i].z, g[i].w}, zw[4] = {z[i].x, z[i].y, z[i].z, z[i].w};
      uint32_t o[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        float2 v = unpack2<T>(gw[k]);
        if constexpr (ACT != kActNone) {
          const float2 d = act_slope<ACT>(unpack2<T>(zw[k]));
          v.x *= d.x, v.y *= d.y;
        }
        sum[2 * k] += v.x, sum[2 * k + 1] += v.y;
        o[k] = pack2<T>(v.x, v.y);
      }
      if (r0 + i < rows) *reinterpret_cast<uint4 *>(dz + (r0 + i) * ld + c) = make_uint4(o[0], o[1], o[2], o[3]); // (ld a multiple of 8)
    }
  }
  if (!bias_sums) return;
#pragma unroll
  for (int k = 0; k < 8; ++k) part[warp][k * 32 + lane] = sum[k];
  __syncthreads();
  const int k = threadIdx.x % 8, l = threadIdx.x / 8; // (neighbouring threads have neighbouring columns)
  const int at = (by * 32 + l) * 8 + k;
  if (at >= ld) return;
  float s = 0.f;
#pragma unroll
  for (int w = 0; w < 8; ++w) s += part[w][k * 32 + l];
  bias_sums[bx * ld + at] = s;
}
// The power of two that brings the largest |v| of the rows that have a label to about 2^13 (1 where nothing finite and
// nonzero is there).  The other rows' dz are zeros, whatever their weights.
__device__ __forceinline__ void find_scale(const float *v, const void *labels, int label_bytes, long long classes, long long n, float *scale, float *tops) {
  float top = 0.f;
#pragma unroll 8
  for (long long i = threadIdx.x; i < n; i += 256) {
    const float a = fabsf(v[i]);
    const long long label = label_at(labels, label_bytes, i);
    if (a < INFINITY && label >= 0 && label < classes) top = fmaxf(top, a);
  }
  for (int d = 16; d; d >>= 1) top = fmaxf(top, __shfl_xor_sync(~0u, top, d));
  if (threadIdx.x % 32 == 0) tops[threadIdx.x / 32] = top;
  __syncthreads();
  if (threadIdx.x) return;
  for (int i = 1; i < 8; ++i) top = fmaxf(top, tops[i]);
  int e = 0;
  if (top > 0.f) frexpf(top, &e);
  *scale = top > 0.f ? ldexpf(1.f, min(max(13 - e, -100), 100)) : 1.f;
}
// What has to be there before a call's products, in one launch: the scale of a loss's gradient, dz of a layer, and
// matrices whose rows do not begin at multiples of 16 bytes copied to where they do (16 bytes a thread).
template <class T> struct PrepareJobs {
  const float *weights; // find_scale
  const void *labels;
  int label_bytes;
  long long num_weights, classes;
  float *scale;
  const T *grad, *pre; // act_grad
  long long ld_grad, ld_pre, ld_dz;
  bool vec_grad, vec_pre;
  T *dz;
  float *bias_sums;
  int rows, cols;
  unsigned row_blocks;
  struct {
    const T *from;
    T *to;
    long long ld_from, ld_to, rows, cols;
  } copy[2];
  unsigned blocks[4]; // of the scale, of dz, of the copies
};
template <class T, int ACT> __global__ void __launch_bounds__(256, 4) tb_dense_prepare_kernel(const __grid_constant__ PrepareJobs<T> jobs) {
  __shared__ float part[8][256];
  after_previous_kernel();
  unsigned b = blockIdx.x;
  if (b < jobs.blocks[0]) return find_scale(jobs.weights, jobs.labels, jobs.label_bytes, jobs.classes, jobs.num_weights, jobs.scale, part[0]);
  b -= jobs.blocks[0];
  if (b < jobs.blocks[1])
    return act_grad<T, ACT>(jobs.grad, jobs.ld_grad, jobs.vec_grad, jobs.pre, jobs.ld_pre, jobs.vec_pre, jobs.dz, jobs.ld_dz, jobs.bias_sums,
                            jobs.rows, jobs.cols, b % jobs.row_blocks, b / jobs.row_blocks, part);
  b -= jobs.blocks[1];
  const int which = b >= jobs.blocks[2];
  if (which) b -= jobs.blocks[2];
  const T *from = which ? jobs.copy[1].from : jobs.copy[0].from;
  T *to = which ? jobs.copy[1].to : jobs.copy[0].to;
  const long long ld_from = which ? jobs.copy[1].ld_from : jobs.copy[0].ld_from, ld_to = which ? jobs.copy[1].ld_to : jobs.copy[0].ld_to;
  const long long rows = which ? jobs.copy[1].rows : jobs.copy[0].rows, cols = which ? jobs.copy[1].cols : jobs.copy[0].cols;
  const long long per = ld_to / 8, i = (long long)b * 256 + threadIdx.x;
  if (i >= rows * per) return;
  const long long r = i / per, c = i % per * 8;
  *reinterpret_cast<uint4 *>(to + r * ld_to + c) = raw8(from + r * ld_from + c, (int)min(8ll, cols - c), false);
}

} // namespace tb
