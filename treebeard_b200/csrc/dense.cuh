// Matrix products on the tensor cores with what follows them fused in:
//   C[m, n] = sum_k A[m, k] B[n, k],  A, B fp16 or bf16, sums in fp32 in tensor memory.
//
// Either operand may lie with k or with its rows one behind the other in memory (the products of the
// backward passes sum over rows): the tensor map's box and the shared-memory descriptor differ, nothing is
// transposed.  A block has one warp that issues the tensor copies, one that issues the matrix instructions
// and eight that take finished tiles out of tensor memory; two accumulators, so that a tile is taken out
// while the next one is computed.  Blocks are persistent and walk over units: a row tile, a run of column
// tiles, a part of the sum.
//
//   PAIR: two blocks of a cluster on one 256 x 256 tile; each brings 128 rows of A and 128 of B, so a stage
//         of 64 k costs an SM 32 KB of L2 traffic for 512 cycles of matrix work (48 KB for one block's 128 x 256).
//   else: one block, 128 x 128 tiles, for products with few tiles.
//
// All waits are bounded: one that gives up ends the launch with a word in tb_dense_status.
#pragma once
#include <cuda.h>
#include <cstdint>
#include "element.cuh"

namespace tb {

constexpr int kDenseThreads = 384, kDenseEndWarps = 8, kDenseK = 64;
constexpr int kDenseStageBytes = 32768, kDenseStages = 6; // 128 rows of A and 128 of B, 64 k each
constexpr int kDenseEndBytes = 4096;                      // a finishing warp's own shared memory
constexpr int kDenseSmem = 1024 + kDenseStages * kDenseStageBytes + kDenseEndWarps * kDenseEndBytes + 256;

__device__ int tb_dense_status; // 0, or 4: a wait gave up

struct DenseProblem {
  CUtensorMap a, b;
  long long M, N;
  int a_rows_inner, b_rows_inner; // 1: rows lie one behind the other, not k
  int m_tiles, n_tiles, k_blocks;
  int chunk, chunks; // column tiles of a unit, units along the columns
  int splits;        // parts of the sum
  int group;         // row tiles that are walked together
  long long units;
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
  asm volatile("{\n .reg .pred p;\n mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n selp.u32 %0, 1, 0, p;\n}"
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
__device__ __forceinline__ void dense_take(uint32_t addr, float (&v)[32]) {
  uint32_t r[32];
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
               "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
                 "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]),
                 "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]),
                 "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
               : "r"(addr));
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
  for (int i = 0; i < 32; ++i) v[i] = __uint_as_float(r[i]);
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
__device__ __forceinline__ DenseUnit dense_unit(const DenseProblem &p, long long u) {
  DenseUnit w;
  w.split = (int)(u % p.splits);
  const long long r = u / p.splits, per = (long long)p.group * p.chunks;
  const int g = (int)(r / per) * p.group, in = (int)(r % per), rows = min(p.group, p.m_tiles - g);
  w.m = g + in % rows;
  w.chunk = in / rows;
  w.n0 = w.chunk * p.chunk;
  w.n1 = min(w.n0 + p.chunk, p.n_tiles);
  w.k0 = (int)((long long)w.split * p.k_blocks / p.splits);
  w.k1 = (int)((long long)(w.split + 1) * p.k_blocks / p.splits);
  return w;
}

// End: what becomes of a tile.  A thread of a finishing warp has one row and 32 columns at a time:
//   start(state, p, row, unit, half)                  once per unit
//   tile(state, p, n, smem)                           once per column tile, n the warp's first column
//   chunk(state, p, v, row, n, smem)                  v[j] = C[row, n + j]; row = the warp's first row + lane
//   stop(state, p, row, unit, half)                   after the unit's last tile
// `half` says which half of a tile's columns the warp has.
template <class T, bool PAIR, class End>
__global__ void __cluster_dims__(PAIR ? 2 : 1, 1, 1) __launch_bounds__(kDenseThreads, 1)
    tb_dense_kernel(const __grid_constant__ DenseProblem p, const __grid_constant__ End end) {
  constexpr int BN = PAIR ? 256 : 128, BM = PAIR ? 256 : 128;
  extern __shared__ unsigned char raw[];
  const uint32_t base = (dense_smem(raw) + 1023u) & ~1023u;
  unsigned char *base_p = raw + (base - dense_smem(raw));
  unsigned char *end_p = base_p + kDenseStages * kDenseStageBytes;
  const uint32_t bars = base + kDenseStages * kDenseStageBytes + kDenseEndWarps * kDenseEndBytes;
  const uint32_t full = bars, empty = bars + 64, tfull = bars + 128, tempty = bars + 144, tmem_at = bars + 160;
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const uint32_t rank = PAIR ? blockIdx.x & 1 : 0;
  const long long first = PAIR ? blockIdx.x >> 1 : blockIdx.x, step = PAIR ? gridDim.x >> 1 : gridDim.x;

  if (warp == 0 && lane == 0) {
    for (int i = 0; i < kDenseStages; ++i) {
      dense_bar_init(full + 8 * i, 1);
      dense_bar_init(empty + 8 * i, 1);
    }
    for (int i = 0; i < 2; ++i) {
      dense_bar_init(tfull + 8 * i, 1);
      dense_bar_init(tempty + 8 * i, kDenseEndWarps * (PAIR ? 2 : 1));
    }
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

  bool ok = true;
  if (warp == 0) {
    if (lane == 0) {
      int stage = 0;
      uint32_t phase = 0;
      long long loads = 0;
      for (long long u = first; ok && u < p.units; u += step) {
        const DenseUnit w = dense_unit(p, u);
        const int row = w.m * BM + (int)rank * 128;
        for (int n = w.n0; ok && n < w.n1; ++n) {
          const int col = n * BN + (int)rank * 128;
          for (int k = w.k0; k < w.k1; ++k) {
            if (!(ok = dense_wait(empty + 8 * stage, phase ^ 1))) break;
            const uint32_t bar = PAIR ? dense_first(full + 8 * stage) : full + 8 * stage;
            if (rank == 0) dense_expect(full + 8 * stage, kDenseStageBytes * (PAIR ? 2 : 1));
            const uint32_t a = base + stage * kDenseStageBytes, b = a + kDenseStageBytes / 2;
            if (p.a_rows_inner) {
              dense_load<PAIR>(a, &p.a, row, k * kDenseK, bar);
              dense_load<PAIR>(a + 8192, &p.a, row + 64, k * kDenseK, bar);
            } else {
              dense_load<PAIR>(a, &p.a, k * kDenseK, row, bar);
            }
            if (p.b_rows_inner) {
              dense_load<PAIR>(b, &p.b, col, k * kDenseK, bar);
              dense_load<PAIR>(b + 8192, &p.b, col + 64, k * kDenseK, bar);
            } else {
              dense_load<PAIR>(b, &p.b, k * kDenseK, col, bar);
            }
            ++loads;
            if (++stage == kDenseStages) stage = 0, phase ^= 1;
          }
        }
      }
      // what was loaded has been used, and every arrival of the matrix unit at this block's barriers is in:
      // the block may end
      for (int i = 0; i < kDenseStages && i < loads; ++i) {
        if (stage-- == 0) stage = kDenseStages - 1, phase ^= 1;
        if (ok) ok = dense_wait(empty + 8 * stage, phase);
        else if (rank == 0) dense_wait(full + 8 * stage, phase); // (copies in flight land before the way out)
      }
    }
  } else if (warp == 1) {
    if (lane == 0 && rank == 0) {
      const uint32_t idesc = 1u << 4 | dense_format<T>() << 7 | dense_format<T>() << 10 | (uint32_t)p.a_rows_inner << 15 |
                             (uint32_t)p.b_rows_inner << 16 | (uint32_t)(BN / 8) << 17 | (uint32_t)(BM / 16) << 24;
      const uint32_t a_step = p.a_rows_inner ? 2048 >> 4 : 32 >> 4, b_step = p.b_rows_inner ? 2048 >> 4 : 32 >> 4;
      int stage = 0, buf = 0;
      uint32_t phase = 0, tphase = 0;
      for (long long u = first; ok && u < p.units; u += step) {
        const DenseUnit w = dense_unit(p, u);
        for (int n = w.n0; ok && n < w.n1; ++n) {
          if (!(ok = dense_wait(tempty + 8 * buf, tphase ^ 1))) break;
          asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
          const uint32_t d = tmem + (uint32_t)(buf * BN);
          for (int k = w.k0; k < w.k1; ++k) {
            if (!(ok = dense_wait(full + 8 * stage, phase))) break;
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            const uint32_t at = base + stage * kDenseStageBytes;
            const uint64_t a = dense_desc(at, p.a_rows_inner), b = dense_desc(at + kDenseStageBytes / 2, p.b_rows_inner);
#pragma unroll
            for (int i = 0; i < kDenseK / 16; ++i) dense_mma<PAIR>(d, a + i * a_step, b + i * b_step, idesc, k > w.k0 || i > 0);
            dense_commit<PAIR>(empty + 8 * stage);
            if (++stage == kDenseStages) stage = 0, phase ^= 1;
          }
          if (!ok) break;
          dense_commit<PAIR>(tfull + 8 * buf);
          if (++buf == 2) buf = 0, tphase ^= 1;
        }
      }
    }
  } else if (warp >= 4) {
    const int e = warp - 4, half = e / 4;
    unsigned char *mine = end_p + e * kDenseEndBytes;
    const uint32_t free_bar = PAIR ? dense_first(tempty) : tempty;
    int buf = 0;
    uint32_t tphase = 0;
    for (long long u = first; ok && u < p.units; u += step) {
      const DenseUnit w = dense_unit(p, u);
      const long long row = (long long)w.m * BM + rank * 128 + (warp % 4) * 32 + lane;
      typename End::State state;
      end.start(state, p, row, w, half);
      for (int n = w.n0; n < w.n1; ++n) {
        const long long col = (long long)n * BN + half * (BN / 2);
        end.tile(state, p, col, mine);
        if (!(ok = __all_sync(~0u, dense_wait(tfull + 8 * buf, tphase)))) break;
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        const uint32_t at = tmem + (uint32_t)(buf * BN + half * (BN / 2)) + ((uint32_t)(warp % 4) << 21);
#pragma unroll 1
        for (int c = 0; c < BN / 64; ++c) {
          float v[32];
          dense_take(at + c * 32, v);
          if (c == BN / 64 - 1) { // the accumulator is free as soon as the last values are in registers
            asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
            if (lane == 0) {
              if constexpr (PAIR)
                asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(free_bar + 8 * buf) : "memory");
              else
                asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(free_bar + 8 * buf) : "memory");
            }
          }
          if (col + c * 32 < p.N) end.chunk(state, p, v, row, col + c * 32, w, mine);
        }
        if (++buf == 2) buf = 0, tphase ^= 1;
      }
      if (ok) end.stop(state, p, row, w, half);
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
constexpr float kLog2e = 1.44269504f, kLn2 = 0.69314718f;

// Phi(z), the integral of the normal distribution, and exp(-z^2 / 2).  erfc's shape after Hastings
// (Approximations for Digital Computers, 1955): Phi(-|z|) = exp(-z^2 / 2) t P(t), t = 1 / (1 + 0.33 |z|);
// P was fitted here, by reweighted least squares, for the relative error: below 1e-6 for all z.  Without
// branches, since a warp's values need both sides of any (the library's erff took most of a layer's time).
__device__ __forceinline__ float normal_integral(float z, float *bell) {
  const float a = fabsf(z), t = inverse_fast(fmaf(a, 0.33f, 1.f));
  float p = fmaf(0.0332859295f, t, -0.105665717f);
  p = fmaf(p, t, 0.067432403f);
  p = fmaf(p, t, 0.0334278586f);
  p = fmaf(p, t, 0.0910052722f);
  p = fmaf(p, t, 0.117216671f);
  p = fmaf(p, t, 0.13164699f);
  p = fmaf(p, t, 0.131651081f);
  *bell = exp2_fast(z * z * (-0.5f * kLog2e));
  const float tail = *bell * t * p;
  return z >= 0.f ? 1.f - tail : tail;
}
__device__ __forceinline__ float act_value(float z, int act) {
  if (act == 1) return z < 0.f ? 0.f : z; // (NaN stays)
  if (act == 2) {
    float bell;
    return z * normal_integral(z, &bell);
  }
  if (act == 3) return z * inverse_fast(1.f + exp2_fast(-kLog2e * z));
  return z;
}
__device__ __forceinline__ float act_slope(float z, int act) {
  if (act == 1) return z > 0.f ? 1.f : 0.f;
  if (act == 2) {
    float bell;
    const float w = normal_integral(z, &bell);
    return fmaf(z * 0.39894228f, bell, w);
  }
  if (act == 3) {
    const float s = inverse_fast(1.f + exp2_fast(-kLog2e * z));
    return s * fmaf(z, 1.f - s, 1.f);
  }
  return 1.f;
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

// Turns 32 rows x 32 columns of a warp around in its shared memory, so that a lane has eight consecutive
// columns of a row: f(row 0..31, column 0, 8, 16 or 24, values).  16-byte pieces are swapped around by the
// row's number, which keeps both directions free of bank conflicts.
template <class F> __device__ __forceinline__ void turned(const float (&v)[32], unsigned char *mine, F f) {
  const int lane = threadIdx.x % 32;
  float4 *s = reinterpret_cast<float4 *>(mine);
#pragma unroll
  for (int i = 0; i < 8; ++i) s[lane * 8 + (i ^ (lane & 7))] = make_float4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]);
  __syncwarp();
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int r = i * 8 + lane / 4, c = lane % 4;
    const float4 x = s[r * 8 + ((2 * c) ^ (r & 7))], y = s[r * 8 + ((2 * c + 1) ^ (r & 7))];
    const float w[8] = {x.x, x.y, x.z, x.w, y.x, y.y, y.z, y.w};
    f(r, c * 8, w);
  }
  __syncwarp();
}

// The same with a lane per column: f(row, value), for results whose rows begin anywhere: a warp then writes 32
// neighbouring elements at a time instead of every eighth.
template <class F> __device__ __forceinline__ void turned_columns(const float (&v)[32], unsigned char *mine, F f) {
  const int lane = threadIdx.x % 32;
  float4 *s = reinterpret_cast<float4 *>(mine);
#pragma unroll
  for (int i = 0; i < 8; ++i) s[lane * 8 + (i ^ (lane & 7))] = make_float4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]);
  __syncwarp();
  const float *w = reinterpret_cast<const float *>(mine) + lane % 4;
#pragma unroll 8
  for (int r = 0; r < 32; ++r) f(r, w[(r * 8 + ((lane / 4) ^ (r & 7))) * 4]);
  __syncwarp();
}

// y = activation(z + bias) + residual, and z + bias
template <class T> struct LinearEnd {
  const T *bias, *residual;
  T *out, *pre;
  long long ld_residual, ld_out, ld_pre;
  int act;
  bool vec_residual, vec_out, vec_pre, vec_bias;
  __device__ __forceinline__ void finish1(float c, long long m, long long n) const {
    const float z = bias ? c + to_float(bias[n]) : c;
    if (pre) pre[m * ld_pre + n] = from_float<T>(z);
    const float y = act_value(z, act);
    out[m * ld_out + n] = from_float<T>(residual ? y + to_float(residual[m * ld_residual + n]) : y);
  }
  __device__ __forceinline__ void finish8(const float (&c)[8], long long m, long long n, long long N) const {
    const int have = (int)min(8ll, N - n);
    float z[8], b[8];
    if (bias) {
      load8(bias + n, b, have, vec_bias);
#pragma unroll
      for (int i = 0; i < 8; ++i) z[i] = c[i] + b[i];
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) z[i] = c[i];
    }
    if (pre) store8(pre + m * ld_pre + n, z, have, vec_pre);
#pragma unroll
    for (int i = 0; i < 8; ++i) z[i] = act_value(z[i], act);
    if (residual) {
      load8(residual + m * ld_residual + n, b, have, vec_residual);
#pragma unroll
      for (int i = 0; i < 8; ++i) z[i] += b[i];
    }
    store8(out + m * ld_out + n, z, have, vec_out);
  }
};

// gradient with respect to an operand: a finished sum, or one piece of it
template <class T> struct SumEnd {
  float *sums; // [rows][ld]: what came before, where the sum comes in pieces
  long long ld;
  T *out;
  const T *skip; // added at the end, or null
  long long ld_out, ld_skip;
  const float *scale; // divides the result; null: 1
  bool first, last, vec_out, vec_skip;
  __device__ __forceinline__ void finish1(float c, long long m, long long n) const {
    float *s = sums + m * ld + n;
    if (!first) c += *s;
    if (!last) {
      *s = c;
      return;
    }
    if (scale) c *= 1.f / *scale;
    out[m * ld_out + n] = from_float<T>(skip ? c + to_float(skip[m * ld_skip + n]) : c);
  }
  __device__ __forceinline__ void finish8(const float (&c)[8], long long m, long long n, long long N) const {
    const int have = (int)min(8ll, N - n);
    float v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = c[i];
    float *s = sums + m * ld + n; // (ld a multiple of 8: whole pieces of 8 are there)
    if (!first) {
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] += s[i];
    }
    if (!last) {
#pragma unroll
      for (int i = 0; i < 8; ++i) s[i] = v[i];
      return;
    }
    if (scale) {
      const float d = 1.f / *scale; // (a power of two)
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] *= d;
    }
    if (skip) {
      float b[8];
      load8(skip + m * ld_skip + n, b, have, vec_skip);
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] += b[i];
    }
    store8(out + m * ld_out + n, v, have, vec_out);
  }
};

// Finishes whole sums in place.
template <class F> struct WholeEnd {
  F f;
  struct State {};
  __device__ __forceinline__ void start(State &, const DenseProblem &, long long, const DenseUnit &, int) const {}
  __device__ __forceinline__ void tile(State &, const DenseProblem &, long long, unsigned char *) const {}
  __device__ __forceinline__ void chunk(State &, const DenseProblem &p, const float (&v)[32], long long row, long long n, const DenseUnit &,
                                        unsigned char *mine) const {
    const long long m0 = row - threadIdx.x % 32;
    if (f.vec_out)
      turned(v, mine, [&](int r, int c, const float (&w)[8]) {
        if (m0 + r < p.M && n + c < p.N) f.finish8(w, m0 + r, n + c, p.N);
      });
    else
      turned_columns(v, mine, [&](int r, float w) {
        if (m0 + r < p.M && n + threadIdx.x % 32 < p.N) f.finish1(w, m0 + r, n + threadIdx.x % 32);
      });
  }
  __device__ __forceinline__ void stop(State &, const DenseProblem &, long long, const DenseUnit &, int) const {}
};
// Keeps the parts of sums that are cut into `splits`: parts[split][row][ld]
struct PartEnd {
  float *parts;
  long long ld;
  struct State {};
  __device__ __forceinline__ void start(State &, const DenseProblem &, long long, const DenseUnit &, int) const {}
  __device__ __forceinline__ void tile(State &, const DenseProblem &, long long, unsigned char *) const {}
  __device__ __forceinline__ void chunk(State &, const DenseProblem &p, const float (&v)[32], long long row, long long n, const DenseUnit &u,
                                        unsigned char *mine) const {
    const long long m0 = row - threadIdx.x % 32;
    turned(v, mine, [&](int r, int c, const float (&w)[8]) {
      if (m0 + r >= p.M || n + c >= p.N) return;
      float4 *d = reinterpret_cast<float4 *>(parts + ((long long)u.split * p.M + m0 + r) * ld + n + c);
      d[0] = make_float4(w[0], w[1], w[2], w[3]);
      d[1] = make_float4(w[4], w[5], w[6], w[7]);
    });
  }
  __device__ __forceinline__ void stop(State &, const DenseProblem &, long long, const DenseUnit &, int) const {}
};
// Adds the parts up, in order, and finishes them.
template <class F>
__global__ void __launch_bounds__(256) tb_dense_join_kernel(const float *parts, int splits, long long ld, long long M, long long N, F f) {
  const long long per = ld / 8, i = (long long)blockIdx.x * 256 + threadIdx.x;
  if (i >= M * per) return;
  const long long m = i / per, n = i % per * 8;
  float v[8] = {};
  for (int s = 0; s < splits; ++s) {
    const float4 *d = reinterpret_cast<const float4 *>(parts + ((long long)s * M + m) * ld + n);
    const float4 a = d[0], b = d[1];
    v[0] += a.x, v[1] += a.y, v[2] += a.z, v[3] += a.w, v[4] += b.x, v[5] += b.y, v[6] += b.z, v[7] += b.w;
  }
  f.finish8(v, m, n, N);
}

__device__ __forceinline__ long long label_at(const void *labels, int bytes, long long m) {
  return bytes == 8 ? static_cast<const long long *>(labels)[m] : static_cast<const int *>(labels)[m];
}
// The biases of a warp's 128 (or 64) columns of a tile in units of log2, in its shared memory; -inf for
// columns behind the last class, which thereby have probability 0.
template <class T, int COLS>
__device__ __forceinline__ void stage_bias(const T *bias, long long n, long long N, float *dst) {
  __syncwarp();
#pragma unroll
  for (int i = threadIdx.x % 32; i < COLS; i += 32) dst[i] = n + i >= N ? -INFINITY : bias ? to_float(bias[n + i]) * kLog2e : 0.f;
  __syncwarp();
}

// Sum of a row's exponentials over the tiles of a unit, relative to the largest score of them, in one pass:
// the sum so far is scaled down whenever a larger score comes.  parts[2 * chunk + half][row]
template <class T, int COLS> struct LseEnd {
  const T *bias;
  const void *labels;
  int label_bytes;
  float2 *parts;
  float *at; // [rows] the label's score
  struct State {
    float top, sum;
    long long label, tile;
  };
  __device__ __forceinline__ void start(State &s, const DenseProblem &p, long long row, const DenseUnit &, int) const {
    s.top = -INFINITY;
    s.sum = 0.f;
    s.label = row < p.M ? label_at(labels, label_bytes, row) : -1;
  }
  __device__ __forceinline__ void tile(State &s, const DenseProblem &p, long long n, unsigned char *mine) const {
    s.tile = n;
    stage_bias<T, COLS>(bias, n, p.N, reinterpret_cast<float *>(mine));
  }
  __device__ __forceinline__ void chunk(State &s, const DenseProblem &p, float (&v)[32], long long row, long long n, const DenseUnit &,
                                        unsigned char *mine) const {
    const long long at_label = s.label - n;
    if (at_label >= 0 && at_label < 32 && s.label < p.N) { // (the score itself, not its multiple)
      float z = 0.f;
#pragma unroll
      for (int j = 0; j < 32; ++j)
        if (j == at_label) z = v[j];
      at[row] = bias ? z + to_float(bias[s.label]) : z;
    }
    const float4 *b4 = reinterpret_cast<const float4 *>(mine) + (n - s.tile) / 4;
    float top = -INFINITY;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float4 b = b4[j];
      v[4 * j] = fmaf(v[4 * j], kLog2e, b.x);
      v[4 * j + 1] = fmaf(v[4 * j + 1], kLog2e, b.y);
      v[4 * j + 2] = fmaf(v[4 * j + 2], kLog2e, b.z);
      v[4 * j + 3] = fmaf(v[4 * j + 3], kLog2e, b.w);
      top = fmaxf(top, fmaxf(fmaxf(v[4 * j], v[4 * j + 1]), fmaxf(v[4 * j + 2], v[4 * j + 3])));
    }
    top = fmaxf(top, s.top);
    const float ref = top == -INFINITY ? 0.f : top; // (all so far forbidden: exponentials are 0)
    float a = 0.f, b = 0.f, c = 0.f, d = 0.f;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      a += exp2_fast(v[4 * j] - ref);
      b += exp2_fast(v[4 * j + 1] - ref);
      c += exp2_fast(v[4 * j + 2] - ref);
      d += exp2_fast(v[4 * j + 3] - ref);
    }
    s.sum = s.sum * exp2_fast(s.top - ref) + ((a + b) + (c + d));
    s.top = top;
  }
  __device__ __forceinline__ void stop(State &s, const DenseProblem &p, long long row, const DenseUnit &u, int half) const {
    if (row < p.M) parts[(2ll * u.chunk + half) * p.M + row] = make_float2(s.top, s.sum);
  }
};
// A row's logarithm and loss from its parts: a lane per row, the parts over the block's warps.
constexpr int kJoinWarps = 8;
__global__ void __launch_bounds__(32 * kJoinWarps) tb_loss_join_kernel(const float2 *parts, int count, const float *at, const void *labels, int label_bytes,
                                                                       long long classes, float *loss, float *lse, long long rows) {
  __shared__ float2 mine[kJoinWarps][32];
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  const long long m = (long long)blockIdx.x * 32 + lane;
  float top = -INFINITY, sum = 0.f;
  auto join = [&](float2 q) {
    const float most = fmaxf(top, q.x), ref = most == -INFINITY ? 0.f : most;
    sum = sum * exp2_fast(top - ref) + q.y * exp2_fast(q.x - ref);
    top = most;
  };
  if (m < rows) {
#pragma unroll 4
    for (int t = warp; t < count; t += kJoinWarps) join(parts[(long long)t * rows + m]);
  }
  mine[warp][lane] = make_float2(top, sum);
  __syncthreads();
  if (warp || m >= rows) return;
#pragma unroll
  for (int w = 1; w < kJoinWarps; ++w) join(mine[w][lane]);
  const float l = fmaf(top == -INFINITY ? 0.f : top, kLn2, logf(sum));
  const long long label = label_at(labels, label_bytes, m);
  lse[m] = l;
  loss[m] = label >= 0 && label < classes ? l - at[m] : 0.f;
}

// dz = weight * (exp(z - lse) - [label]) * scale, rounded, and the sums of its columns over 32 rows before
// that: bias_sums[row / 32][ld]
template <class T, int COLS> struct ScoreGradEnd {
  const T *bias; // of the piece's first class
  const void *labels;
  int label_bytes;
  const float *grad, *lse, *scale;
  T *dz;
  long long ld, first, classes; // class of column 0, all classes
  float *bias_sums;
  struct State {
    float weight, lse2;
    long long label, tile;
  };
  __device__ __forceinline__ void start(State &s, const DenseProblem &p, long long row, const DenseUnit &, int) const {
    s.weight = s.lse2 = 0.f;
    s.label = -1;
    if (row >= p.M) return;
    const long long label = label_at(labels, label_bytes, row);
    if (label < 0 || label >= classes) return; // (its dz are zeros whatever the scores)
    s.label = label - first;
    s.weight = grad[row] * *scale;
    s.lse2 = lse[row] * kLog2e;
  }
  __device__ __forceinline__ void tile(State &s, const DenseProblem &p, long long n, unsigned char *mine) const {
    s.tile = n;
    stage_bias<T, COLS>(bias, n, p.N, reinterpret_cast<float *>(mine + 2048));
  }
  __device__ __forceinline__ void chunk(State &s, const DenseProblem &p, float (&v)[32], long long row, long long n, const DenseUnit &,
                                        unsigned char *mine) const {
    const int lane = threadIdx.x % 32;
    const float4 *b4 = reinterpret_cast<const float4 *>(mine + 2048) + (n - s.tile) / 4;
    const bool live = s.weight != 0.f;
    const float lse2 = s.lse2;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float4 b = b4[j];
      v[4 * j] = s.weight * exp2_fast(fmaf(v[4 * j], kLog2e, b.x - lse2));
      v[4 * j + 1] = s.weight * exp2_fast(fmaf(v[4 * j + 1], kLog2e, b.y - lse2));
      v[4 * j + 2] = s.weight * exp2_fast(fmaf(v[4 * j + 2], kLog2e, b.z - lse2));
      v[4 * j + 3] = s.weight * exp2_fast(fmaf(v[4 * j + 3], kLog2e, b.w - lse2));
    }
    if (!live) {
#pragma unroll
      for (int j = 0; j < 32; ++j) v[j] = 0.f;
    }
    const long long at = s.label - n;
    if (live && at >= 0 && at < 32) {
#pragma unroll
      for (int j = 0; j < 32; ++j)
        if (j == at) v[j] -= s.weight;
    }
    uint4 *q = reinterpret_cast<uint4 *>(mine);
#pragma unroll
    for (int i = 0; i < 4; ++i)
      q[lane * 4 + (i ^ ((lane >> 1) & 3))] = make_uint4(pack2<T>(v[8 * i], v[8 * i + 1]), pack2<T>(v[8 * i + 2], v[8 * i + 3]),
                                                         pack2<T>(v[8 * i + 4], v[8 * i + 5]), pack2<T>(v[8 * i + 6], v[8 * i + 7]));
    __syncwarp();
    const long long m0 = row - lane;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int r = i * 8 + lane / 4, c = lane % 4;
      if (m0 + r < p.M && n + c * 8 < ld) *reinterpret_cast<uint4 *>(dz + (m0 + r) * ld + n + c * 8) = q[r * 4 + (c ^ ((r >> 1) & 3))];
    }
    __syncwarp();
    if (bias_sums) {
      // sums over the 32 lanes of 32 values each: every step halves the values and doubles the lanes summed
#pragma unroll
      for (int d = 16; d; d >>= 1) {
        const bool upper = lane & d;
#pragma unroll
        for (int j = 0; j < d; ++j) {
          const float keep = upper ? v[j + d] : v[j], give = upper ? v[j] : v[j + d];
          v[j] = keep + __shfl_xor_sync(~0u, give, d);
        }
      }
      if (m0 < p.M && n + lane < ld) bias_sums[m0 / 32 * ld + n + lane] = v[0];
    }
  }
  __device__ __forceinline__ void stop(State &, const DenseProblem &, long long, const DenseUnit &, int) const {}
};

// dz = grad * activation'(pre), rounded; sums of its columns over 32 rows before that.  32 rows x 256 columns
// a block, four rows a warp, whose loads are under way together.
template <class T>
__global__ void __launch_bounds__(256) tb_act_grad_kernel(const T *grad, long long ld_grad, bool vec_grad, const T *pre, long long ld_pre,
                                                          bool vec_pre, int act, T *dz, long long ld, float *bias_sums, long long rows,
                                                          long long cols) {
  __shared__ float part[8][256];
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  const long long c = ((long long)blockIdx.y * 32 + lane) * 8, r0 = (long long)blockIdx.x * 32 + warp * 4;
  const int have = (int)min(8ll, cols - c);
  float g[4][8], z[4][8], sum[8] = {};
  if (have > 0) {
#pragma unroll
    for (int i = 0; i < 4; ++i) load8(grad + (r0 + i) * ld_grad + c, g[i], r0 + i < rows ? have : 0, vec_grad);
    if (act) {
#pragma unroll
      for (int i = 0; i < 4; ++i) load8(pre + (r0 + i) * ld_pre + c, z[i], r0 + i < rows ? have : 0, vec_pre);
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int k = 0; k < 8; ++k) g[i][k] *= act_slope(z[i][k], act);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (r0 + i >= rows) break;
      store8(dz + (r0 + i) * ld + c, g[i], 8, true); // (ld a multiple of 8)
#pragma unroll
      for (int k = 0; k < 8; ++k) sum[k] += g[i][k];
    }
  }
  if (!bias_sums) return;
#pragma unroll
  for (int k = 0; k < 8; ++k) part[warp][k * 32 + lane] = sum[k];
  __syncthreads();
  const int k = threadIdx.x % 8, l = threadIdx.x / 8; // (neighbouring threads have neighbouring columns)
  const long long at = ((long long)blockIdx.y * 32 + l) * 8 + k;
  if (at >= ld) return;
  float s = 0.f;
#pragma unroll
  for (int w = 0; w < 8; ++w) s += part[w][k * 32 + l];
  bias_sums[blockIdx.x * ld + at] = s;
}

// out[c] = sum over `count` rows of sums[., c], times 1 / scale: eight warps take every eighth row each
template <class T>
__global__ void __launch_bounds__(256) tb_column_sum_kernel(const float *sums, long long count, long long ld, T *out, long long cols, const float *scale) {
  __shared__ float part[8][32];
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  const long long c = (long long)blockIdx.x * 32 + lane;
  float s = 0.f;
  if (c < cols)
    for (long long t = warp; t < count; t += 8) s += sums[t * ld + c];
  part[warp][lane] = s;
  __syncthreads();
  if (warp || c >= cols) return;
  for (int i = 1; i < 8; ++i) s += part[i][lane];
  out[c] = from_float<T>(scale ? s / *scale : s);
}

// The power of two that brings the largest |v| to about 2^13 (1 where nothing finite and nonzero is there).
__global__ void __launch_bounds__(1024) tb_scale_kernel(const float *v, long long n, float *scale) {
  __shared__ float tops[32];
  float top = 0.f;
  for (long long i = threadIdx.x; i < n; i += 1024)
    if (fabsf(v[i]) < INFINITY) top = fmaxf(top, fabsf(v[i]));
  for (int d = 16; d; d >>= 1) top = fmaxf(top, __shfl_xor_sync(~0u, top, d));
  if (threadIdx.x % 32 == 0) tops[threadIdx.x / 32] = top;
  __syncthreads();
  if (threadIdx.x) return;
  for (int i = 1; i < 32; ++i) top = fmaxf(top, tops[i]);
  int e = 0;
  if (top > 0.f) frexpf(top, &e);
  *scale = top > 0.f ? ldexpf(1.f, min(max(13 - e, -100), 100)) : 1.f;
}

// A matrix whose rows do not begin at multiples of 16 bytes, copied to where they do: 16 bytes a thread.
template <class T>
__global__ void __launch_bounds__(256) tb_align_rows_kernel(const T *src, long long ld_src, T *dst, long long ld, long long rows, long long cols) {
  const long long per = ld / 8, all = rows * per;
  for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < all; i += (long long)gridDim.x * 256) {
    const long long r = i / per, c = i % per * 8;
    uint32_t w[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const unsigned short *p = reinterpret_cast<const unsigned short *>(src + r * ld_src + c + 2 * k);
      w[k] = (c + 2 * k < cols ? __ldg(p) : 0) | (uint32_t)(c + 2 * k + 1 < cols ? __ldg(p + 1) : 0) << 16;
    }
    *reinterpret_cast<uint4 *>(dst + r * ld + c) = make_uint4(w[0], w[1], w[2], w[3]);
  }
}

} // namespace tb
