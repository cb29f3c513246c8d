// Products of block tensors: D[M, N] = A[M, K] . B[N, K]^T, both operands E4M3
// with one power-of-two scale per row and 128 columns (block_scale.cuh).
//
//   D[m, n] = sum_b 2^(ea[m, b] + eb[n, b]) sum_{k in block b} A[m, k] B[n, k]
//
// tcgen05.mma kind::mxf8f6f4 applies the scales inside the tensor core (its
// scale factors cover 32 columns; the four instructions of a 128-column slab
// name the same scale byte), so the accumulator is never read back during the
// reduction and the scales cost four bytes per row and 512 columns. The MMA
// takes the scales from tensor memory; one tcgen05.cp per 128 rows brings
// those of four slabs there, 512 bytes, in the order the cast stored them.
//
// Two kernels:
//
// split_kernel  one 128 x BN tile (BN 16, 32 or 64) on one CTA, the reduction
//   split over the CTAs of a cluster, whose partial tiles meet in distributed
//   shared memory and are added in rank order. For problems with too few
//   256 x 256 tiles to fill the GPU: with few tokens (swapped: the 128 side
//   holds the weight's rows) it is bound by reading the weight, and S CTAs per
//   tile keep every SM's loads in flight; for a small weight gradient over
//   many tokens the split is what fills the SMs. No workspace, no atomics: the
//   result does not depend on timing. For up to 16 tokens it can cast them
//   itself (QX): every CTA casts its slabs of the few rows again, which costs
//   less than a kernel of its own before it. Measured: 1 x 4096 x 4096 8.2 us
//   (a 16.8 MB weight, cast of x included), 61 x 1024 x 4096 9.6 us with the
//   cast's launch before it; tiles 5.3 us + 0.36 per slab.
//
// pair_kernel  256 x 256 tiles on CTA pairs (tcgen05 cta_group::2), persistent,
//   for everything large: bound by the tensor cores. Two accumulators of 256
//   columns fill tensor memory, which leaves none for the scales, so they
//   overlap by 24 columns, the room of two sets of scales: the next tile's MMAs
//   start as soon as the epilogue has read the shared columns, which it reads
//   first. Measured: 8192 x 4096 x
//   4096 (bf16 out) 106 us, 2.6 PFLOP/s, and 33 us with a reduction of 1024. A
//   slab takes 634 cycles where the MMAs alone take 512: per slab an SM's shared
//   memory takes in 32 KB and gives 48 KB (A's own rows, all of B) to the MMA,
//   640 cycles at 128 bytes each. With eight slabs a tile it is 720, as the
//   epilogue's staging passes there too, and 13 % of the time the operands are
//   late: L2 delivers 13 TB/s. A long run is held to 1.3 GHz by the power limit.
//   Handing over a tile costs 130 cycles, copying scales 1.5 %, a scaled MMA
//   4 % over a plain one.
#include <cuda.h>
#include <cmath>
#include "block_scale.cuh"
#include "tcgen05.cuh"

namespace apa {
int num_sms();
namespace blk {

using gemm::BM;
using gemm::kSlab;
using gemm::fence_after;
using gemm::fence_before;
using gemm::fu;
using gemm::mbar_expect_tx;
using gemm::mbar_init;
using gemm::mbar_wait;
using gemm::sdesc;
using gemm::smem_u32;
using gemm::tma_load_2d;

struct OutArgs {
  void* out; int64_t ldo; int out_dt;
  const void* bias; int bias_dt;      // [N], added in fp32 (nullable)
  int accumulate;                     // fp32 out: add to it
  int vec;                            // rows of out are 16-byte aligned
  int M, N;                           // of the caller's D
};

// Instruction descriptor of kind::mxf8f6f4: E4M3 x E4M3, E8M0 scales (bit 23),
// N >> 3 at bit 17, M >> 7 at bit 27; the scale byte of B at bit 4 and of A at
// bit 29 are or-ed in per slab.
template <int BN, int TM>
__host__ __device__ constexpr uint32_t mx_idesc() {
  return ((uint32_t)(BN >> 3) << 17) | (1u << 23) | ((uint32_t)(TM >> 7) << 27);
}

template <bool PAIR>
__device__ __forceinline__ void mx_mma(uint32_t d, uint64_t a, uint64_t b, uint32_t id, uint32_t sfa, uint32_t sfb,
                                       uint32_t accumulate) {
  if constexpr (PAIR) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %6, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::mxf8f6f4.block_scale.scale_vec::1X [%0], %1, %2, %3, [%4], [%5], p;\n\t}" ::"r"(
            d),
        "l"(a), "l"(b), "r"(id), "r"(sfa), "r"(sfb), "r"(accumulate));
  } else {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %6, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::mxf8f6f4.block_scale.scale_vec::1X [%0], %1, %2, %3, [%4], [%5], p;\n\t}" ::"r"(
            d),
        "l"(a), "l"(b), "r"(id), "r"(sfa), "r"(sfb), "r"(accumulate));
  }
}

// 512 bytes of scales (32 rows of 16 bytes, no swizzle: 8-row groups 128 bytes
// apart) to four tensor-memory columns, repeated in every lane quarter.
__device__ __forceinline__ uint64_t scale_desc(uint32_t saddr) {
  return (uint64_t)((saddr >> 4) & 0x3FFFu) | ((uint64_t)1 << 16) | ((uint64_t)(128 >> 4) << 32) | ((uint64_t)1 << 46);
}

__device__ __forceinline__ void prefetch_map(const CUtensorMap* tm) {
  asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(tm)) : "memory");
}

template <bool PAIR>
__device__ __forceinline__ void scale_copy(uint32_t taddr, uint32_t saddr) {
  if constexpr (PAIR)
    asm volatile("tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(scale_desc(saddr)) : "memory");
  else
    asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(scale_desc(saddr)) : "memory");
}

__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint32_t* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, "
      "[%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr));
}

// Four neighbouring elements of one output row: bias, accumulation, rounding.
// vec: the row's addresses allow one store.
__device__ __forceinline__ void put4(const OutArgs& o, int m, int n, float4 x) {
  float v[4] = {x.x, x.y, x.z, x.w};
  const int64_t at = (int64_t)m * o.ldo + n;
  const int c = min(4, o.N - n);
  if (o.bias) {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (j < c) v[j] += to_f32(o.bias, o.bias_dt, n + j);
  }
  if (o.vec && c == 4) {
    if (o.out_dt == APA_DT_F32) {
      float4* d = reinterpret_cast<float4*>(static_cast<float*>(o.out) + at);
      if (o.accumulate) {
        const float4 y = *d;
        v[0] += y.x; v[1] += y.y; v[2] += y.z; v[3] += y.w;
      }
      *d = make_float4(v[0], v[1], v[2], v[3]);
    } else {
      uint2 w;
      if (o.out_dt == APA_DT_BF16) w = make_uint2(bf16x2(v[0], v[1]), bf16x2(v[2], v[3]));
      else w = make_uint2(f16x2_from_f32(v[0], v[1]), f16x2_from_f32(v[2], v[3]));
      *reinterpret_cast<uint2*>(static_cast<uint16_t*>(o.out) + at) = w;
    }
    return;
  }
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    if (j < c) {
      if (o.accumulate) v[j] += static_cast<const float*>(o.out)[at + j];
      from_f32(o.out, o.out_dt, at + j, v[j]);
    }
  }
}

// ---------------------------------------------------------------------------
// split_kernel
// ---------------------------------------------------------------------------
template <int BN> struct SplitCfg {
  static constexpr int kABytes = BM * kSlab;
  static constexpr int kBBytes = BN * kSlab;
  static constexpr int kScaleBytes = 1024;          // 512 of A, 512 of B
  static constexpr int kStageBytes = kABytes + kBBytes;
  // two CTAs per SM: one loads while the other finishes
  static constexpr int kStages = BN == 64 ? 4 : 5;
  static constexpr int kTmemCols = BN == 64 ? 128 : BN == 32 ? 64 : 32;
  static constexpr int kSmemBytes = kStages * (kStageBytes + kScaleBytes) + 1024 + 256;
  static constexpr int kThreads = 192;
  static_assert((BN + 4) * BM * 4 <= kStages * kStageBytes, "the tile reuses the stages");
  static_assert(BN + 8 <= kTmemCols, "tensor memory");
  static_assert(2 * (kSmemBytes + 1024) <= 228 * 1024, "two CTAs per SM");
};

// Rows of the BN side as they come, to be cast by the kernel (QX).
struct RowArgs { const void* x; int64_t ld; int dt, vec; int64_t K; };

struct SplitArgs {
  int rows_a, rows_b;       // rows of the 128 side and of the BN side
  int tiles_b;
  int kb_count;             // 128-column slabs
  int split;                // CTAs per tile (cluster size)
  int swap;                 // the 128 side is D's N
  RowArgs rows;             // QX
  OutArgs o;
};

template <int BN, bool QX>
__global__ void __launch_bounds__(192, 2)
    split_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB,
                 const __grid_constant__ CUtensorMap tmSA, const __grid_constant__ CUtensorMap tmSB, SplitArgs p) {
  using C = SplitCfg<BN>;
  constexpr int kStages = C::kStages;
  pdl_launch_dependents();
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  uint8_t* smA = smem;
  uint8_t* smB = smem + kStages * C::kABytes;
  uint8_t* smS = smem + kStages * C::kStageBytes;
  uint64_t* full = reinterpret_cast<uint64_t*>(smS + kStages * C::kScaleBytes);
  uint64_t* empty = full + kStages;
  uint64_t* done = empty + kStages;
  uint64_t* cast = done + 1;               // QX: the stage's rows are cast
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(cast + kStages);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int tile = blockIdx.x / p.split, rank = blockIdx.x - tile * p.split;
  const int a0 = (tile / p.tiles_b) * BM, b0 = (tile % p.tiles_b) * BN;
  // slabs of this rank; split <= kb_count, so none is empty
  const int kb0 = (int)((int64_t)p.kb_count * rank / p.split);
  const int kb1 = (int)((int64_t)p.kb_count * (rank + 1) / p.split);

  if (threadIdx.x == 0) {
    for (int s = 0; s < kStages; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
      mbar_init(&cast[s], 128);
    }
    mbar_init(done, 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)),
                 "r"((uint32_t)C::kTmemCols)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  if (threadIdx.x == 32 * 2) {
    prefetch_map(&tmA);
    prefetch_map(&tmB);
    prefetch_map(&tmSA);
    prefetch_map(&tmSB);
  }
  fence_before();
  __syncthreads();
  fence_after();
  const uint32_t tmem = *tmem_slot;
  const uint32_t sfa = tmem + BN, sfb = tmem + BN + 4;
  pdl_wait();

  if (warp == 0) {
    if (lane == 0) {
      int stage = 0;
      uint32_t phase = 0;
      bool ok = true;
      for (int kb = kb0; kb < kb1; ++kb) {
        if (!mbar_wait(&empty[stage], phase ^ 1u, kStatusTimeoutEmpty)) { ok = false; break; }
        const bool scales = kb == kb0 || (kb & 3) == 0;
        mbar_expect_tx(&full[stage], QX ? C::kABytes + (scales ? 512 : 0)
                                        : C::kStageBytes + (scales ? C::kScaleBytes : 0));
        tma_load_2d(smA + stage * C::kABytes, &tmA, kb * kSlab, a0, &full[stage]);
        if constexpr (!QX) tma_load_2d(smB + stage * C::kBBytes, &tmB, kb * kSlab, b0, &full[stage]);
        if (scales) {
          uint8_t* s = smS + stage * C::kScaleBytes;
          tma_load_2d(s, &tmSA, a0, kb >> 2, &full[stage]);
          if constexpr (!QX) tma_load_2d(s + 512, &tmSB, b0 & ~127, kb >> 2, &full[stage]);
        }
        if (++stage == kStages) { stage = 0; phase ^= 1u; }
      }
      (void)ok;
    }
    __syncwarp();
  } else if (warp == 1) {
    if (lane == 0) {
      int stage = 0;
      uint32_t phase = 0;
      bool ok = true;
      // rows b0 .. of a chunk of 128 start at scale column (b0 % 128) / 32: 0
      // or, for the second tile of 64 rows, 2 (an odd column faults)
      const uint32_t sfb0 = sfb + (uint32_t)((b0 & 127) >> 5);
      for (int kb = kb0; kb < kb1; ++kb) {
        if (!mbar_wait(&full[stage], phase, kStatusTimeoutFull)) { ok = false; break; }
        if (QX && !mbar_wait(&cast[stage], phase, kStatusTimeoutFull)) { ok = false; break; }
        fence_after();
        const uint32_t s = smem_u32(smS + stage * C::kScaleBytes);
        const bool scales = kb == kb0 || (kb & 3) == 0;
        if (scales) scale_copy<false>(sfa, s);
        if (QX || scales) scale_copy<false>(sfb, s + 512);
        const uint32_t j = (uint32_t)(kb & 3);
        // rows cast here have their slab's scale in byte 0
        const uint32_t id = mx_idesc<BN, BM>() | ((QX ? 0u : j) << 4) | (j << 29);
        const uint32_t a = smem_u32(smA + stage * C::kABytes), b = smem_u32(smB + stage * C::kBBytes);
#pragma unroll
        for (int k = 0; k < 4; ++k)
          mx_mma<false>(tmem, sdesc(a + 32 * k), sdesc(b + 32 * k), id, sfa, sfb0, (kb != kb0 || k != 0) ? 1u : 0u);
        gemm::mma_commit<false>(&empty[stage]);
        if (++stage == kStages) { stage = 0; phase ^= 1u; }
      }
      if (ok) gemm::mma_commit<false>(done);
    }
    __syncwarp();
  }

  if constexpr (QX) {
    // warps 2 .. 5 cast the rows, slab by slab, into the swizzled layout that
    // TMA would have written: sixteen threads a row, eight columns each, rows
    // rr and rr + 8; the loads of four slabs are under way together. Rows past
    // the last stay as they are: they make columns that nothing reads.
    static_assert(BN == 16, "two rows per thread");
    if (warp >= 2) {
      const int t = threadIdx.x - 64, g = t & 15, rr = t >> 4;
      const RowArgs& x = p.rows;
      int stage = 0;
      uint32_t phase = 0;
      bool ok = true;
      for (int base = kb0; ok && base < kb1; base += 4) {
        float v[4][2][8];
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const int64_t c0 = (int64_t)(base + i) * kSlab + 8 * g;
            const int n = base + i < kb1 && rr + 8 * h < p.rows_b ? (int)max((int64_t)0, min((int64_t)8, x.K - c0)) : 0;
            load8(x.x, x.dt, (rr + 8 * h) * x.ld + c0, n, x.vec && n == 8, v[i][h]);
          }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          if (base + i >= kb1) break;
          // one lane's verdict for the warp: shuffles follow
          bool free = true;
          if (lane == 0) free = mbar_wait(&empty[stage], phase ^ 1u, kStatusTimeoutEmpty);
          ok = __shfl_sync(0xFFFFFFFFu, free ? 1 : 0, 0) != 0;
          if (!ok) break;
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            if (8 * h >= p.rows_b) break;             // no second row anywhere
            float (&y)[8] = v[i][h];
            auto top = [&]() {
              float a = 0.0f;
#pragma unroll
              for (int j = 0; j < 8; j += 2) a = max_abs(y[j], y[j + 1], a);
              return a;
            };
            float a = top();
            if (is_inf(a)) {
#pragma unroll
              for (int j = 0; j < 8; ++j) y[j] = inf_to_nan(y[j]);
              a = top();
            }
            uint32_t m = __float_as_uint(a);
#pragma unroll
            for (int o = 8; o > 0; o >>= 1) m = max(m, __shfl_xor_sync(0xFFFFFFFFu, m, o));
            const uint32_t b = scale_byte(m);
            uint8_t* row = smB + stage * C::kBBytes + h * 1024 + rr * 128;
            *reinterpret_cast<uint2*>(row + (((g >> 1) ^ rr) << 4) + (g & 1) * 8) = codes8(y, inv_scale(b));
            if (g == 0) *reinterpret_cast<uint32_t*>(smS + stage * C::kScaleBytes + 512 + (rr + 8 * h) * 16) = b;
          }
          gemm::fence_async_smem();
          gemm::mbar_arrive(&cast[stage]);
          if (++stage == kStages) { stage = 0; phase ^= 1u; }
        }
      }
      __syncwarp();
    }
  }

  // epilogue: warps 2 .. 5 read the accumulator's lane quarter warp % 4
  const int q = warp & 3;
  bool ready = false;
  if (warp >= 2) {
    if (lane == 0) ready = mbar_wait(done, 0, kStatusTimeoutAcc);
    ready = __shfl_sync(0xFFFFFFFFu, ready ? 1 : 0, 0) != 0;
    fence_after();
  }
  const uint32_t lanes = tmem + ((uint32_t)(q * 32) << 16);
  constexpr int kC = BN >= 32 ? 32 : 16;
  // The tile goes through shared memory in the output's order, over the
  // operand stages (every load has landed and every MMA has read it once
  // `done` completes): [128][BN + 4], or [BN][128] when swapped. Both orders
  // are written and read without bank conflicts.
  float* part = reinterpret_cast<float*>(smem);
  if (warp >= 2 && ready) {
#pragma unroll 1
    for (int c = 0; c < BN; c += kC) {
      if (b0 + c >= p.rows_b) break;
      uint32_t r[kC];
      if constexpr (kC == 32) gemm::tmem_ld32_nowait(lanes + c, r);
      else tmem_ld16(lanes + c, r);
      gemm::tmem_wait_ld();
      if (p.swap) {
#pragma unroll
        for (int j = 0; j < kC; ++j) part[(c + j) * BM + q * 32 + lane] = fu(r[j]);
      } else {
        float4* d = reinterpret_cast<float4*>(part + (q * 32 + lane) * (BN + 4) + c);
#pragma unroll
        for (int j = 0; j < kC / 4; ++j)
          d[j] = make_float4(fu(r[4 * j]), fu(r[4 * j + 1]), fu(r[4 * j + 2]), fu(r[4 * j + 3]));
      }
    }
  }
  __syncwarp();
  if (p.split == 1) __syncthreads();
  else gemm::cluster_sync();
  if (warp >= 2 && ready) {
    // units of four elements along the output's rows, the ranks' shares one
    // after the other; a unit's partials are added in rank order
    const int outer = p.swap ? min(BN, p.rows_b - b0) : min(BM, p.rows_a - a0);
    const int per = p.swap ? BM / 4 : BN / 4;
    const int pitch = p.swap ? BM : BN + 4;
    const int m0 = p.swap ? b0 : a0, n0 = p.swap ? a0 : b0;
    const int units = outer * per;
    const int u1 = units * (rank + 1) / p.split;
    for (int u = units * rank / p.split + (int)threadIdx.x - 64; u < u1; u += 128) {
      const int i = u / per, j = u - i * per;
      if (n0 + 4 * j >= p.o.N) continue;
      const float* at = part + i * pitch + 4 * j;
      float4 x;
      if (p.split == 1) {
        x = *reinterpret_cast<const float4*>(at);
      } else {
        float4 y[8];
#pragma unroll
        for (int s = 0; s < 8; ++s) {
          if (s < p.split) {
            const uint32_t a = gemm::map_to_cta(at, (uint32_t)s);
            asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
                         : "=f"(y[s].x), "=f"(y[s].y), "=f"(y[s].z), "=f"(y[s].w)
                         : "r"(a));
          }
        }
        x = y[0];
#pragma unroll
        for (int s = 1; s < 8; ++s) {
          if (s < p.split) { x.x += y[s].x; x.y += y[s].y; x.z += y[s].z; x.w += y[s].w; }
        }
      }
      put4(p.o, m0 + i, n0 + 4 * j, x);
    }
  }
  __syncwarp();
  if (p.split > 1) gemm::cluster_sync();   // no CTA leaves while another reads its partials
  fence_before();
  __syncthreads();
  fence_after();
  if (warp == 1)
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"((uint32_t)C::kTmemCols)
                 : "memory");
}

// ---------------------------------------------------------------------------
// pair_kernel
// ---------------------------------------------------------------------------
// Arrive on a barrier of either CTA of the pair. CTA scope: what is handed
// over is tensor memory, ordered by the tcgen05 fences on both sides; a
// cluster-scope release would flush this thread's ordinary stores first, in
// the path between two tiles.
__device__ __forceinline__ void arrive_peer(uint32_t cluster_addr) {
  asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(cluster_addr) : "memory");
}

constexpr int kEpiBox = 4096;      // one staging buffer: 32 rows x 128 bytes
constexpr int kAccStride = 232;    // second accumulator: columns 232 .. 487
// two sets of scales, used in turn, so that copying the next one does not wait
// for the MMAs that still read the last: 4 columns of A's and 8 of B's each
constexpr int kPairScales = 488, kScaleSet = 12;
static_assert(kAccStride + 256 <= kPairScales && kPairScales + 2 * kScaleSet <= 512, "tensor memory");
static_assert(256 - kAccStride <= 64, "the shared columns are read with the epilogue's first unit");

template <int EW> struct PairCfg {
  static constexpr int kTile = 256;
  static constexpr int kHalfBytes = BM * kSlab;                 // this CTA's rows of A, and of B
  static constexpr int kStageBytes = 2 * kHalfBytes;
  static constexpr int kScaleBytes = 512 + 1024;                // own 128 rows of A, all 256 of B
  static constexpr int kBoxes = EW == 4 ? 1 : 2;                // staging buffers per epilogue warp
  static constexpr int kStages = EW == 4 ? 6 : 4;
  static constexpr int kWarpCols = 1024 / EW;                   // columns per epilogue warp
  static constexpr int kUnits = kWarpCols / 64;
  static constexpr int kThreads = 64 + 32 * EW;
  static constexpr int kSmemBytes =
      kStages * (kStageBytes + kScaleBytes) + EW * (kBoxes * kEpiBox + kWarpCols * 4) + 256 + 1024;
  static_assert(kSmemBytes <= 232448, "shared memory");
};

// One product of a launch.
struct Problem {
  int kb_count;
  int splits;           // the reduction is split over this many units per tile
  int slice_rows;       // rows of one split's slice of the workspace (out is the workspace when splits > 1)
  int chunk;            // slabs accumulated at once; later chunks are added to out
  int tma_out;          // out written by TMA stores (or reductions)
  OutArgs o;
};

struct ProblemMaps { CUtensorMap a, b, sa, sb, o; };

// Column sums of [parts, cols] fp32 partials (a bias gradient's, which the cast
// of the gradient left), added in order and rounded once. In this launch they
// save their own: a step of 1111 x 520 x 1000 takes 33.5 us with, 37 without,
// 16384 x 384 x 1536 89.8 and 91.1.
struct ColumnSums { const float* part; int parts, cols; void* out; int out_dt; };

// NP products in one launch. Units (tile, split) go round the CTA pairs. With
// two products, `units0` units of the first, the longer ones, are dealt first;
// they may end in the middle of a round, so the pairs from `late` on, which
// have one unit less, take `extra` units of the second product each before
// all go on with what is left.
template <int NP> struct PairArgs {
  Problem q[NP];
  int units0, units1, late, extra;
  ColumnSums sums;
};
template <int NP> struct PairMaps { ProblemMaps m[NP]; };

// One pass of the schedule: slabs kb0 .. kb1 of an output tile. A unit's
// chunks follow each other on the same pair.
struct Pass {
  int prob, unit, phase;            // phase 0, 1, 2: first product, extra units, the rest; 3: done
  int tile, split, first, kb0, kb1, end;
};

template <int NP>
__device__ __forceinline__ void pass_unit(const PairArgs<NP>& p, Pass& a) {
  const Problem& q = p.q[NP == 1 ? 0 : a.prob];
  a.tile = a.unit;
  a.split = 0;
  a.first = 0;
  a.end = q.kb_count;
  if (q.splits > 1) {
    // kb_count < 2^24 and splits < 2^7: 32 bits hold the products
    a.tile = a.unit / q.splits;
    a.split = a.unit - a.tile * q.splits;
    a.first = (int)((uint32_t)q.kb_count * (uint32_t)a.split / (uint32_t)q.splits);
    a.end = (int)((uint32_t)q.kb_count * (uint32_t)(a.split + 1) / (uint32_t)q.splits);
  }
  a.kb0 = a.first;
  a.kb1 = min(a.kb0 + q.chunk, a.end);
}

// The unit at a.unit of the current phase, or of the first phase after it that
// has one for this pair.
template <int NP>
__device__ __forceinline__ void pass_settle(const PairArgs<NP>& p, int pair, int step, Pass& a) {
  if (a.phase == 0) {
    if (a.unit < p.units0) return pass_unit(p, a);
    if (NP == 1) { a.phase = 3; return; }
    a.prob = 1;
    a.phase = 1;
    a.unit = pair - p.late;
  }
  const int dealt = p.extra * (step - p.late);
  if (a.phase == 1) {
    if (a.unit >= 0 && a.unit < min(dealt, p.units1)) return pass_unit(p, a);
    a.phase = 2;
    a.unit = dealt + pair;
  }
  if (a.unit < p.units1) return pass_unit(p, a);
  a.phase = 3;
}

template <int NP>
__device__ __forceinline__ void pass_first(const PairArgs<NP>& p, int pair, int step, Pass& a) {
  a.prob = 0;
  a.phase = 0;
  a.unit = pair;
  pass_settle(p, pair, step, a);
}

template <int NP>
__device__ __forceinline__ void pass_next(const PairArgs<NP>& p, int pair, int step, Pass& a) {
  if (a.kb1 < a.end) {
    a.kb0 = a.kb1;
    a.kb1 = min(a.kb0 + p.q[NP == 1 ? 0 : a.prob].chunk, a.end);
    return;
  }
  a.unit += a.phase == 1 ? step - p.late : step;
  pass_settle(p, pair, step, a);
}

// A staged fp32 box added to out. Each element of out is added to by one warp,
// in its program order, so the result does not depend on timing.
__device__ __forceinline__ void tma_add_2d(const CUtensorMap* tm, const void* src, int x, int y) {
  asm volatile("cp.reduce.async.bulk.tensor.2d.global.shared::cta.add.tile.bulk_group [%0, {%2, %3}], [%1];" ::"l"(
                   reinterpret_cast<uint64_t>(tm)),
               "r"(smem_u32(src)), "r"(x), "r"(y)
               : "memory");
}

// A staged box (32 rows of 128 bytes, 128-byte swizzle) to rows that TMA
// cannot store to (unaligned, or a ragged last 16 bytes): one row per step,
// one 4-byte word per lane, so a warp's store covers whole lines.
__device__ __forceinline__ void put_box(const OutArgs& o, const uint8_t* box, int lane, int row0, int col0,
                                        bool add) {
  const bool out16 = o.out_dt != APA_DT_F32;
  const int rows = min(32, o.M - row0);
  const int col = col0 + (out16 ? 2 * lane : lane);
#pragma unroll 4
  for (int r = 0; r < rows; ++r) {
    const uint32_t w =
        *reinterpret_cast<const uint32_t*>(box + r * 128 + (((lane >> 2) ^ (r & 7)) << 4) + (lane & 3) * 4);
    const int64_t at = (int64_t)(row0 + r) * o.ldo + col;
    if (out16) {
      uint16_t* d = static_cast<uint16_t*>(o.out) + at;
      if (col + 1 < o.N && (reinterpret_cast<uintptr_t>(d) & 3u) == 0) {
        *reinterpret_cast<uint32_t*>(d) = w;
      } else {
        if (col < o.N) d[0] = (uint16_t)w;
        if (col + 1 < o.N) d[1] = (uint16_t)(w >> 16);
      }
    } else if (col < o.N) {
      float* d = static_cast<float*>(o.out) + at;
      *d = add ? *d + fu(w) : fu(w);
    }
  }
}

template <int EW, int NP>
__global__ void __launch_bounds__(64 + 32 * EW, 1)
    pair_kernel(const __grid_constant__ PairMaps<NP> maps, const __grid_constant__ PairArgs<NP> p) {
  using C = PairCfg<EW>;
  constexpr int kStages = C::kStages;
  pdl_launch_dependents();
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  uint8_t* smA = smem;
  uint8_t* smB = smem + kStages * C::kHalfBytes;
  uint8_t* smE = smem + kStages * C::kStageBytes;                         // staging boxes, 128-byte swizzled
  uint8_t* smS = smE + EW * C::kBoxes * kEpiBox;
  float* smBias = reinterpret_cast<float*>(smS + kStages * C::kScaleBytes);
  uint64_t* full = reinterpret_cast<uint64_t*>(smBias + EW * C::kWarpCols);
  uint64_t* empty = full + kStages;
  uint64_t* tfull = empty + kStages;
  uint64_t* tempty = tfull + 2;
  uint64_t* tshared = tempty + 2;          // the overlapping columns of the current tile have been read
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(tshared + 1);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = gemm::cluster_rank();
  const int pair = (int)(blockIdx.x >> 1), step = (int)(gridDim.x >> 1);
  auto coords = [&](const Problem& q, int tile, int& mb, int& nb) {
    gemm::tile_coords(tile, (q.o.M + 255) / 256, (q.o.N + 255) / 256, gemm::kGroupM / 2, mb, nb);
  };

  if (threadIdx.x == 0) {
    for (int s = 0; s < kStages; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int a = 0; a < 2; ++a) {
      mbar_init(&tfull[a], 1);
      mbar_init(&tempty[a], EW * 2);
    }
    mbar_init(tshared, 4 * 2);             // four warps of each CTA hold those columns
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)),
                 "r"(512u)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  }
  if (threadIdx.x >= 32 * 2 && threadIdx.x < 32 * 2 + NP) {
    const ProblemMaps& m = maps.m[threadIdx.x - 32 * 2];
    prefetch_map(&m.a);
    prefetch_map(&m.b);
    prefetch_map(&m.sa);
    prefetch_map(&m.sb);
    prefetch_map(&m.o);
  }
  fence_before();
  gemm::cluster_sync();
  fence_after();
  const uint32_t tmem = *tmem_slot;
  pdl_wait();

  if (warp == 0) {
    if (lane == 0) {
      int stage = 0;
      uint32_t phase = 0;
      bool ok = true;
      Pass a;
      for (pass_first(p, pair, step, a); ok && a.phase < 3; pass_next(p, pair, step, a)) {
        const ProblemMaps& m = maps.m[NP == 1 ? 0 : a.prob];
        int mb, nb;
        coords(p.q[NP == 1 ? 0 : a.prob], a.tile, mb, nb);
        const int a_row = mb * 256 + (int)rank * BM, b_row = nb * 256 + (int)rank * BM;
        for (int kb = a.kb0; kb < a.kb1; ++kb) {
          if (!mbar_wait(&empty[stage], phase ^ 1u, kStatusTimeoutEmpty)) { ok = false; break; }
          const bool scales = kb == a.kb0 || (kb & 3) == 0;
          // the even CTA's barrier expects both CTAs' bytes
          if (rank == 0) mbar_expect_tx(&full[stage], 2 * (C::kStageBytes + (scales ? C::kScaleBytes : 0)));
          const uint32_t bar = gemm::map_to_cta(&full[stage], 0);
          gemm::tma_load_2d_pair(smA + stage * C::kHalfBytes, &m.a, kb * kSlab, a_row, bar);
          gemm::tma_load_2d_pair(smB + stage * C::kHalfBytes, &m.b, kb * kSlab, b_row, bar);
          if (scales) {
            uint8_t* s = smS + stage * C::kScaleBytes;
            gemm::tma_load_2d_pair(s, &m.sa, a_row, kb >> 2, bar);
            gemm::tma_load_2d_pair(s + 512, &m.sb, nb * 256, kb >> 2, bar);
          }
          if (++stage == kStages) { stage = 0; phase ^= 1u; }
        }
      }
      // until the MMAs have released every stage
      for (int i = 0; ok && i < kStages; ++i) {
        if (!mbar_wait(&empty[stage], phase ^ 1u, kStatusTimeoutEmpty)) ok = false;
        if (++stage == kStages) { stage = 0; phase ^= 1u; }
      }
    }
    __syncwarp();
  } else if (warp == 1) {
    if (lane == 0 && rank == 0) {
      int stage = 0, local = 0;
      uint32_t phase = 0;
      bool ok = true;
      uint32_t set = 0;
      Pass a;
      for (pass_first(p, pair, step, a); ok && a.phase < 3; pass_next(p, pair, step, a), ++local) {
        const int acc = local & 1;
        if (!mbar_wait(&tempty[acc], ((uint32_t)(local >> 1) & 1u) ^ 1u, kStatusTimeoutAcc)) { ok = false; break; }
        // the previous tile's shared columns
        if (local > 0 && !mbar_wait(tshared, (uint32_t)(local - 1) & 1u, kStatusTimeoutAcc)) { ok = false; break; }
        fence_after();
        const uint32_t d = tmem + (uint32_t)(acc * kAccStride);
        for (int kb = a.kb0; kb < a.kb1; ++kb) {
          if (!mbar_wait(&full[stage], phase, kStatusTimeoutFull)) { ok = false; break; }
          fence_after();
          const uint32_t j = (uint32_t)(kb & 3);
          const bool scales = kb == a.kb0 || j == 0;
          if (scales) set ^= 1u;
          const uint32_t sfa = tmem + kPairScales + set * kScaleSet, sfb = sfa + 4;
          if (scales) {
            const uint32_t s = smem_u32(smS + stage * C::kScaleBytes);
            scale_copy<true>(sfa, s);
            scale_copy<true>(sfb, s + 512);
            scale_copy<true>(sfb + 4, s + 1024);
          }
          const uint32_t id = mx_idesc<256, 256>() | (j << 4) | (j << 29);
          const uint32_t sa = smem_u32(smA + stage * C::kHalfBytes), sb = smem_u32(smB + stage * C::kHalfBytes);
#pragma unroll
          for (int k = 0; k < 4; ++k)
            mx_mma<true>(d, sdesc(sa + 32 * k), sdesc(sb + 32 * k), id, sfa, sfb, (kb != a.kb0 || k != 0) ? 1u : 0u);
          gemm::mma_commit<true>(&empty[stage]);
          if (++stage == kStages) { stage = 0; phase ^= 1u; }
        }
        if (ok) gemm::mma_commit<true>(&tfull[acc]);
      }
    }
    __syncwarp();
  } else {
    const int q = warp & 3, e = warp - 2, part = e >> 2;
    uint8_t* boxes = smE + e * C::kBoxes * kEpiBox;
    float* sb = smBias + e * C::kWarpCols;
    if constexpr (NP == 2) {
      // done while the first tile is under way; sixteen loads at a time
      if (p.sums.part != nullptr) {
        const ColumnSums& t = p.sums;
        // 64 bits: the last step passes 2^31 where cols is near it
        for (int64_t c = ((int)blockIdx.x * EW + e) * 32 + lane; c < t.cols; c += (int)gridDim.x * EW * 32) {
          float x = 0.0f;
          for (int r = 0; r < t.parts; r += 16) {
            float v[16];
#pragma unroll
            for (int k = 0; k < 16; ++k) v[k] = r + k < t.parts ? __ldcg(t.part + (int64_t)(r + k) * t.cols + c) : 0.0f;
#pragma unroll
            for (int k = 0; k < 16; ++k) x += v[k];
          }
          from_f32(t.out, t.out_dt, c, x);
        }
      }
    }
    int local = 0;
    int slot = 0, inflight = 0;           // staging ring; TMA stores that may still read their box
    const uint32_t te0 = gemm::map_to_cta(&tempty[0], 0), te1 = gemm::map_to_cta(&tempty[1], 0);
    const uint32_t ts = gemm::map_to_cta(tshared, 0);
    auto arrive = [&](uint32_t bar) {
      fence_before();
      __syncwarp();
      if (lane == 0) arrive_peer(bar);
    };
    Pass a;
    for (pass_first(p, pair, step, a); a.phase < 3; pass_next(p, pair, step, a), ++local) {
      const Problem& prob = p.q[NP == 1 ? 0 : a.prob];
      const OutArgs& o = prob.o;
      const CUtensorMap* tmO = &maps.m[NP == 1 ? 0 : a.prob].o;
      const bool out16 = o.out_dt != APA_DT_F32;
      int mb, nb;
      coords(prob, a.tile, mb, nb);
      const int acc = local & 1;
      const int row0 = mb * 256 + (int)rank * BM + q * 32;
      const int orow = row0 + a.split * prob.slice_rows;
      const int col_base = nb * 256 + part * C::kWarpCols;
      // a unit's later chunks, and all of an accumulating product, are added to out
      const bool later = a.kb0 != a.first;
      const bool add = later || o.accumulate;
      const bool bias = o.bias != nullptr && !later;
      if (bias) {
        __syncwarp();
        for (int c = lane; c < C::kWarpCols; c += 32)
          sb[c] = col_base + c < o.N ? to_f32(o.bias, o.bias_dt, col_base + c) : 0.0f;
        __syncwarp();
      }
      bool ready = true;
      if (lane == 0) ready = mbar_wait(&tfull[acc], (uint32_t)(local >> 1) & 1u, kStatusTimeoutAcc);
      ready = __shfl_sync(0xFFFFFFFFu, ready ? 1 : 0, 0) != 0;
      if (!ready) break;
      fence_after();
      if (later && inflight > 0) {
        // the earlier chunk's stores must have landed, not just left
        if (lane == 0) gemm::bulk_wait_all();
        __syncwarp();
        inflight = 0;
        slot = 0;
      }
      const uint32_t tb = tmem + ((uint32_t)(q * 32) << 16) + (uint32_t)(acc * kAccStride + part * C::kWarpCols);
      // the columns the two accumulators share are the last of the first one
      // and the first of the second: those go first
      const int shared_part = acc == 0 ? EW / 4 - 1 : 0;
#pragma unroll 1
      for (int i = 0; i < C::kUnits; ++i) {
        const int u = acc == 0 ? C::kUnits - 1 - i : i;
        const int col0 = col_base + u * 64;
        uint32_t r[64];
        gemm::tmem_ld32_nowait(tb + (uint32_t)(u * 64), r);
        gemm::tmem_ld32_nowait(tb + (uint32_t)(u * 64 + 32), r + 32);
        gemm::tmem_wait_ld();
        if (i == 0 && part == shared_part) arrive(ts);
        if (i == C::kUnits - 1) arrive(acc ? te1 : te0);
        if (col0 >= o.N || row0 >= o.M) continue;      // warp-uniform
        if (bias) {
#pragma unroll
          for (int c = 0; c < 16; ++c) {
            const float4 b = reinterpret_cast<const float4*>(sb + u * 64)[c];
            gemm::add2(r[4 * c], r[4 * c + 1], b.x, b.y);
            gemm::add2(r[4 * c + 2], r[4 * c + 3], b.z, b.w);
          }
        }
        if (out16) {
          if (o.out_dt == APA_DT_BF16) {
#pragma unroll
            for (int k = 0; k < 32; ++k) r[k] = bf16x2(fu(r[2 * k]), fu(r[2 * k + 1]));
          } else {
#pragma unroll
            for (int k = 0; k < 32; ++k) r[k] = f16x2_from_f32(fu(r[2 * k]), fu(r[2 * k + 1]));
          }
        }
#pragma unroll
        for (int b = 0; b < 2; ++b) {
          const int x = col0 + 32 * b;
          if ((out16 && b == 1) || x >= o.N) break;
          uint8_t* box = boxes + slot * kEpiBox;
          if (inflight == C::kBoxes) {
            if (lane == 0) gemm::bulk_wait_read<C::kBoxes - 1>();
            --inflight;
          }
          __syncwarp();
          gemm::stage_row(box, lane, r + 32 * b);
          if (prob.tma_out) {
            gemm::fence_async_smem();
            __syncwarp();
            if (lane == 0) {
              if (add) tma_add_2d(tmO, box, x, orow);
              else gemm::tma_store_2d(tmO, box, x, orow);
              gemm::bulk_commit();
            }
            ++inflight;
            slot = slot + 1 == C::kBoxes ? 0 : slot + 1;
          } else {
            __syncwarp();
            put_box(o, box, lane, row0, x, add);
          }
        }
      }
    }
    if (inflight > 0 && lane == 0) gemm::bulk_wait_all();
    __syncwarp();
  }

  // neither CTA leaves while the other may signal its barriers or read its tensor memory
  fence_before();
  gemm::cluster_sync();
  fence_after();
  if (warp == 1)
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
}

// ---------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------
// E4M3 operand: dims {K, rows}, box {128, box_rows}, 128-byte swizzle, zeros
// past the edges.
int code_map(CUtensorMap* tm, const void* p, int64_t rows, int64_t K, int64_t ld, int box_rows) {
  gemm::EncodeFn enc = gemm::get_encode();
  if (!enc) return APA_ERR_CUDA;
  cuuint64_t dims[2] = {(cuuint64_t)K, (cuuint64_t)rows};
  cuuint64_t strides[1] = {(cuuint64_t)ld};
  cuuint32_t box[2] = {(cuuint32_t)kSlab, (cuuint32_t)box_rows};
  cuuint32_t one[2] = {1, 1};
  return enc(tm, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(p), dims, strides, box, one,
             CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
             CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS ? APA_OK : APA_ERR_CUDA;
}

// Scale words: dims {rows_pad, groups of four blocks}, box {box_words, 1}.
int scale_map(CUtensorMap* tm, const void* p, int64_t rows, int64_t kb_count, int box_words) {
  gemm::EncodeFn enc = gemm::get_encode();
  if (!enc) return APA_ERR_CUDA;
  const int64_t rp = rows_padded(rows);
  cuuint64_t dims[2] = {(cuuint64_t)rp, (cuuint64_t)((kb_count + 3) / 4)};
  cuuint64_t strides[1] = {(cuuint64_t)(rp * 4)};
  cuuint32_t box[2] = {(cuuint32_t)box_words, 1};
  cuuint32_t one[2] = {1, 1};
  return enc(tm, CU_TENSOR_MAP_DATA_TYPE_UINT32, 2, const_cast<void*>(p), dims, strides, box, one,
             CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_NONE,
             CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS ? APA_OK : APA_ERR_CUDA;
}

int64_t cdiv64(int64_t a, int64_t b) { return (a + b - 1) / b; }

struct Operand { const void* q; int64_t ld; const void* sc; int64_t rows; };

// B's codes and scales are not read with `rows` (QX).
template <int BN, bool QX = false>
int launch_split(const Operand& A, const Operand& B, int64_t K, const OutArgs& o, bool swap, int split,
                 cudaStream_t s, const RowArgs& rows = RowArgs{}) {
  using C = SplitCfg<BN>;
  static unsigned long long attr = 0;
  if (int st = allow_smem(split_kernel<BN, QX>, C::kSmemBytes, &attr)) return st;
  const int64_t kb = (K + kSlab - 1) / kSlab;
  CUtensorMap ta, tb, tsa, tsb;
  if (int st = code_map(&ta, A.q, A.rows, K, A.ld, BM)) return st;
  if (int st = scale_map(&tsa, A.sc, A.rows, kb, 128)) return st;
  tb = ta;
  tsb = tsa;
  if constexpr (!QX) {
    if (int st = code_map(&tb, B.q, B.rows, K, B.ld, BN)) return st;
    if (int st = scale_map(&tsb, B.sc, B.rows, kb, 128)) return st;
  }
  SplitArgs p;
  p.rows_a = (int)A.rows; p.rows_b = (int)B.rows;
  p.tiles_b = (int)((B.rows + BN - 1) / BN);
  p.kb_count = (int)kb; p.split = split; p.swap = swap ? 1 : 0; p.rows = rows; p.o = o;
  const int64_t grid = (A.rows + BM - 1) / BM * p.tiles_b * split;
  if (grid > (1ll << 31) - 1) return APA_ERR_INVALID;
  return launch_kernel(split_kernel<BN, QX>, dim3((unsigned)grid), dim3(C::kThreads), C::kSmemBytes, s, split, ta, tb,
                       tsa, tsb, p) == cudaSuccess ? APA_OK : APA_ERR_CUDA;
}

// Output: dims {N, M}, box {128 bytes, 32 rows}, 128-byte swizzle.
int out_map(CUtensorMap* tm, const OutArgs& o, int64_t rows) {
  gemm::EncodeFn enc = gemm::get_encode();
  if (!enc) return APA_ERR_CUDA;
  const int es = elem_bytes(o.out_dt);
  const CUtensorMapDataType dt = o.out_dt == APA_DT_F32   ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
                                 : o.out_dt == APA_DT_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16
                                                          : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
  cuuint64_t dims[2] = {(cuuint64_t)o.N, (cuuint64_t)rows};
  cuuint64_t strides[1] = {(cuuint64_t)(o.ldo * es)};
  cuuint32_t box[2] = {(cuuint32_t)(128 / es), 32};
  cuuint32_t one[2] = {1, 1};
  return enc(tm, dt, 2, o.out, dims, strides, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
             CU_TENSOR_MAP_L2_PROMOTION_NONE, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS ? APA_OK
                                                                                                 : APA_ERR_CUDA;
}

// CTA pairs of the kernel that run at once on the current device (0: none).
template <int EW, int NP>
int pair_slots() {
  using C = PairCfg<EW>;
  static unsigned long long attr = 0;
  static int slots[64];        // per device; written before its bit of `known`
  static unsigned long long known = 0;
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return 0;
  dev &= 63;
  if (__atomic_load_n(&known, __ATOMIC_ACQUIRE) >> dev & 1ull) return slots[dev];
  if (allow_smem(pair_kernel<EW, NP>, C::kSmemBytes, &attr)) return 0;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(2 * num_sms(), 1, 1);
  cfg.blockDim = dim3(C::kThreads, 1, 1);
  cfg.dynamicSmemBytes = C::kSmemBytes;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = 2;
  at[0].val.clusterDim.y = 1;
  at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  int n = 0;
  if (cudaOccupancyMaxActiveClusters(&n, pair_kernel<EW, NP>, &cfg) != cudaSuccess) {
    (void)cudaGetLastError();
    n = 0;
  }
  slots[dev] = n;
  __atomic_fetch_or(&known, 1ull << dev, __ATOMIC_RELEASE);
  return n;
}

// The slices of a split product: fp32, rows padded to whole tiles (a store's
// box never reaches into the next slice), columns to 16 bytes.
int64_t slice_rows(int64_t M) { return cdiv64(M, 256) * 256; }
int64_t slice_ld(int64_t N) { return (N + 3) / 4 * 4; }
int64_t split_bytes(int64_t M, int64_t N, int splits) {
  return splits > 1 ? splits * slice_rows(M) * slice_ld(N) * 4 : 0;
}

struct SumArgs { const float* ws; int64_t slice, ld; int splits; OutArgs o; };

// Adds the slices in order, then bias, accumulation and rounding.
__global__ void __launch_bounds__(256) block_sum_kernel(SumArgs p) {
  pdl_launch_dependents();
  pdl_wait();
  const int per = (int)(p.ld / 4);
  const int64_t total = (int64_t)p.o.M * per;
  for (int64_t e = (int64_t)blockIdx.x * 256 + threadIdx.x; e < total; e += (int64_t)gridDim.x * 256) {
    const int m = (int)(e / per), n = (int)(e - (int64_t)m * per) * 4;
    const float4* at = reinterpret_cast<const float4*>(p.ws + (int64_t)m * p.ld + n);
    float4 x = __ldcg(at);
    for (int s = 1; s < p.splits; s += 4) {
      float4 y[4];
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (s + k < p.splits) y[k] = __ldcg(at + (int64_t)(s + k) * p.slice / 4);
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (s + k < p.splits) { x.x += y[k].x; x.y += y[k].y; x.z += y[k].z; x.w += y[k].w; }
    }
    put4(p.o, m, n, x);
  }
}

// Slabs accumulated at once for an fp32 output. The tensor core drops the bits
// that the running sum cannot hold instead of rounding them, so the error grows
// with the length of the chain (measured against 64 bits: 5e-7 of the result
// after 8192 columns, 3e-6 after 32768, where rounded chunks stay below 5e-7).
// A 16-bit output's own rounding is a thousand times that.
constexpr int kChunkSlabs = 64;

// Maps and arguments of one product; its slices lie in ws when it is split.
int fill_problem(const Operand& A, const Operand& B, int64_t K, OutArgs o, int splits, void* ws, ProblemMaps* m,
                 Problem* q) {
  const int64_t kb = (K + kSlab - 1) / kSlab;
  if (int st = code_map(&m->a, A.q, A.rows, K, A.ld, BM)) return st;
  if (int st = code_map(&m->b, B.q, B.rows, K, B.ld, BM)) return st;
  if (int st = scale_map(&m->sa, A.sc, A.rows, kb, 128)) return st;
  if (int st = scale_map(&m->sb, B.sc, B.rows, kb, 256)) return st;
  q->kb_count = (int)kb; q->splits = splits; q->slice_rows = 0;
  int64_t out_rows = o.M;
  if (splits > 1) {
    out_rows = slice_rows(o.M) * splits;
    if (out_rows > (1ll << 31) - 1) return APA_ERR_INVALID;
    q->slice_rows = (int)slice_rows(o.M);
    o.out = ws; o.ldo = slice_ld(o.N); o.out_dt = APA_DT_F32; o.bias = nullptr; o.accumulate = 0; o.vec = 1;
    o.N = (int)o.ldo;
  }
  // only an fp32 output can be added to
  q->chunk = o.out_dt == APA_DT_F32 ? kChunkSlabs : (int)kb;
  q->o = o;
  // a TMA store writes whole 16-byte pieces, past N too where N ends inside one
  q->tma_out = o.vec && ((int64_t)o.N * elem_bytes(o.out_dt)) % 16 == 0;
  m->o = m->a;
  if (q->tma_out)
    if (int st = out_map(&m->o, o, out_rows)) return st;
  return APA_OK;
}

// The second kernel of a split product.
int launch_sum(const OutArgs& o, int splits, const void* ws, cudaStream_t s) {
  const int64_t ld = slice_ld(o.N);
  const SumArgs q{static_cast<const float*>(ws), slice_rows(o.M) * ld, ld, splits, o};
  const int64_t blocks = cdiv64(o.M * (ld / 4), 256);
  return launch_kernel(block_sum_kernel, dim3((unsigned)std::min<int64_t>(blocks, 8 * num_sms())), dim3(256), 0, s, 1,
                       q) == cudaSuccess ? APA_OK : APA_ERR_CUDA;
}

// A unit's time in slabs, two of them to hand a tile over. Where TMA cannot store
// the rows, a tile takes twelve for its epilogue at least (both gradients of
// 100000 x 100 x 100 74 us, counted by slabs alone 97). A floor of six for the
// other tiles, their epilogue's time, made the split too coarse: 512 x 4096 x
// 4096 35 us against 31.
int64_t unit_cost(int64_t slabs, bool tma_out) { return (tma_out ? slabs : std::max<int64_t>(slabs, 12)) + 2; }

int64_t pair_units(const OutArgs& o, int splits) { return cdiv64(o.M, 256) * cdiv64(o.N, 256) * splits; }

template <int EW, int NP>
int launch_pairs(const PairMaps<NP>& maps, PairArgs<NP>& p, int64_t units0, int64_t units1, cudaStream_t s) {
  using C = PairCfg<EW>;
  int slots = pair_slots<EW, NP>();
  if (slots < 1) return APA_ERR_UNSUPPORTED;
  if (g_gemm_sm_limit > 0) slots = std::max(1, std::min(slots, g_gemm_sm_limit / 2));
  if (units0 + units1 > (1ll << 31) - 1 - 4 * (int64_t)num_sms()) return APA_ERR_INVALID;
  const int pairs = (int)std::min<int64_t>(units0 + units1, slots);
  p.units0 = (int)units0; p.units1 = (int)units1;
  p.late = 0; p.extra = 0;
  if (NP == 2) {
    // how many of the second product's units a unit of the first is worth
    const Problem &a = p.q[0], &b = p.q[NP - 1];
    const int64_t c0 = unit_cost(cdiv64(a.kb_count, a.splits), a.tma_out), c1 = unit_cost(b.kb_count, b.tma_out);
    p.late = (int)(units0 % pairs);
    const int64_t worth = std::max<int64_t>(1, (2 * c0 + c1) / (2 * c1));
    p.extra = p.late ? (int)std::min(worth, cdiv64(units1, pairs - p.late)) : 0;
  }
  return launch_kernel(pair_kernel<EW, NP>, dim3(2 * pairs), dim3(C::kThreads), C::kSmemBytes, s, 2, maps, p) ==
                 cudaSuccess ? APA_OK : APA_ERR_CUDA;
}

template <int EW>
int launch_pair(const Operand& A, const Operand& B, int64_t K, const OutArgs& o, int splits, void* ws, cudaStream_t s) {
  PairMaps<1> m;
  PairArgs<1> p;
  p.sums = ColumnSums{};
  if (int st = fill_problem(A, B, K, o, splits, ws, &m.m[0], &p.q[0])) return st;
  if (int st = launch_pairs<EW, 1>(m, p, pair_units(o, splits), 0, s)) return st;
  return splits > 1 ? launch_sum(o, splits, ws, s) : APA_OK;
}

// kind 0: split_kernel with `bn`, `split` and `swap`; 1: pair_kernel with `ew`
// epilogue warps and `split` units per tile.
struct BlockPlan { int kind, bn, split, swap, ew; };

// The faster of both kernels by a model fitted to timings on a B200 (us, back
// to back). A 128 x 64 tile costs 5.3 + 0.36 per slab in each round of two
// CTAs per SM, and its cluster 0.9, or 2.2 for eight CTAs on more than one
// CTA per SM; clusters of four and eight leave an eighth of the slots empty.
// A 256 x 256 tile costs 0.8 + 0.44 per slab in each wave of CTA pairs, after
// 3 to start; the slices of a split product 3 for the second kernel and their
// bytes at 12 TB/s (they stay in L2). Rows that TMA cannot store to cost the
// pair 3.5 per wave. Both sides of the choice: 512 x 1024 x 4096 9.1 on tiles
// of 64 (split 4), 11.7 on pairs; 512 x 1536 x 33280 44.7 (split 4 of 128 x 128
// tiles) and 30.7.
BlockPlan block_plan(int64_t M, int64_t N, int64_t K, bool aligned) {
  const int64_t kb = cdiv64(K, kSlab);
  const int64_t small = std::min(M, N), big = std::max(M, N);
  BlockPlan best{0, 0, 1, M <= N ? 1 : 0, 8};
  best.bn = small <= 16 ? 16 : small <= 32 ? 32 : 64;
  const int64_t tiles = cdiv64(big, BM) * cdiv64(small, best.bn);
  double cost = 1e30;
  for (int split = 1; split <= 8 && split <= kb; split *= 2) {
    const int64_t ctas = tiles * split;
    const double rounds = std::ceil((double)ctas / ((split > 2 ? 1.75 : 2.0) * num_sms()));
    const double share = split == 1 ? 0.0 : split == 8 && ctas > num_sms() ? 2.2 : 0.9;
    const double t = rounds * (5.3 + 0.36 * (double)cdiv64(kb, split) + share);
    if (t < cost) { cost = t; best.split = split; }
  }
  const int64_t pt = cdiv64(M, 256) * cdiv64(N, 256);
  const int64_t pairs = std::max(1, num_sms() / 2);
  for (int split = 1; split <= 64 && split <= kb; ++split) {
    // a split pays where units would leave pairs idle, in whole waves
    if (split > 1 && pt * split > 2 * pairs) break;
    const double waves = (double)cdiv64(pt * split, pairs);
    const int64_t slabs = cdiv64(kb, split);
    double t = 3.0 + waves * (0.8 + 0.44 * (double)slabs + (aligned || split > 1 ? 0.0 : 3.5));
    if (split > 1) t += 3.0 + 8.0 * (double)split * (double)M * (double)N / 12e6;
    if (t < cost) {
      cost = t;
      // eight warps where the epilogue is exposed (one wave, few slabs, slow
      // stores), else four and a deeper ring: 8192 x 4096 x 4096 107 against
      // 111 us, 33280 x 1536 x 512 37 against 33
      best = BlockPlan{1, 0, split, 0, slabs < 8 || waves <= 1.0 || !aligned ? 8 : 4};
    }
  }
  return best;
}

// A caller's choice (APA_BLOCK_*): the automatic plan stands where it is 0.
int force_plan(int code, int64_t M, int64_t N, int64_t K, BlockPlan* p) {
  if (code == APA_BLOCK_AUTO) return APA_OK;
  const int bn = code & 0x7F, split = (code >> 7) & 0x7F, swap = (code >> 14) & 1, ew = (code >> 15) & 0xF;
  if (code < 0 || (code >> 19) != 0 || split < 1) return APA_ERR_INVALID;
  if (split > cdiv64(K, kSlab)) return APA_ERR_INVALID;      // no unit without a slab
  if (bn == 0) {
    if ((ew != 4 && ew != 8) || swap) return APA_ERR_INVALID;
    p->kind = 1;
  } else {
    if ((bn != 16 && bn != 32 && bn != 64) || split > 8 || ew != 0) return APA_ERR_INVALID;
    // the MMA takes scales from even columns of tensor memory only, 64 rows
    // apart: narrower tiles are for a side of one tile
    if (bn < 64 && (swap ? M : N) > bn) return APA_ERR_INVALID;
    p->kind = 0;
  }
  p->bn = bn; p->split = split; p->swap = swap; p->ew = ew;
  return APA_OK;
}

int block_gemm(const Operand& A, const Operand& B, int64_t K, const OutArgs& o, const BlockPlan& p, void* ws,
               cudaStream_t s) {
  if (p.kind == 1)
    return p.ew == 8 ? launch_pair<8>(A, B, K, o, p.split, ws, s) : launch_pair<4>(A, B, K, o, p.split, ws, s);
  const Operand& x = p.swap ? B : A;
  const Operand& y = p.swap ? A : B;
  switch (p.bn) {
    case 16: return launch_split<16>(x, y, K, o, p.swap, p.split, s);
    case 32: return launch_split<32>(x, y, K, o, p.swap, p.split, s);
    default: return launch_split<64>(x, y, K, o, p.swap, p.split, s);
  }
}

// Two products in one launch, the first with units at least as long as the
// second's: a backward's weight gradient and input gradient, which read
// different casts of the same gradient. One launch less, and the second fills
// the CTA pairs that the first leaves idle in its last round (4096 x 4096 over
// 8192 tokens: 256 and 512 tiles on 74 pairs; the training step of that layer
// takes 392 us with both in one launch, 410 with two; the casts and both
// gradients alone, in one launch and in two: 1 x 4096 x 4096 29.5 and 31, 512 x
// 4096 x 4096 31 and 44, 16384 x 384 x 1536 58 and 66, 33280 x 512 x 512 49 and
// 58). The first is split when a tile of it would take longer than an even share
// of all the work.
int dual_split(const OutArgs& o0, int64_t K0, const OutArgs& o1, int64_t K1) {
  const int64_t pairs = std::max(1, num_sms() / 2);
  const int64_t kb0 = cdiv64(K0, kSlab), kb1 = cdiv64(K1, kSlab);
  const auto tma = [](const OutArgs& o) { return (int64_t)o.N * elem_bytes(o.out_dt) % 16 == 0; };
  const int64_t c0 = unit_cost(kb0, tma(o0)), c1 = unit_cost(kb1, tma(o1));
  const int64_t work = pair_units(o0, 1) * c0 + pair_units(o1, 1) * c1;
  const int64_t share = std::max<int64_t>(cdiv64(work, pairs), c1);
  // a split unit of less than eight slabs costs more to add than it gains
  return (int)std::max<int64_t>(1, std::min(std::min(cdiv64(c0, share), kb0 / 8), (int64_t)64));
}

// Whether the launch's epilogue warps can add `parts` rows of column sums
// before their first tile is done: a row costs them 100 cycles, a slab 634.
bool dual_adds(int64_t parts, int64_t K0, int split) { return parts <= 4 * cdiv64(cdiv64(K0, kSlab), split); }

int block_gemm_dual(const Operand& A0, const Operand& B0, int64_t K0, const OutArgs& o0, const Operand& A1,
                    const Operand& B1, int64_t K1, const OutArgs& o1, const ColumnSums& sums, int split, void* ws,
                    cudaStream_t s) {
  PairMaps<2> m;
  PairArgs<2> p;
  p.sums = sums;
  if (int st = fill_problem(A0, B0, K0, o0, split, ws, &m.m[0], &p.q[0])) return st;
  if (int st = fill_problem(A1, B1, K1, o1, 1, nullptr, &m.m[1], &p.q[1])) return st;
  const int64_t u0 = pair_units(o0, split), u1 = pair_units(o1, 1);
  // as in block_plan: eight epilogue warps for few slabs or a single round
  const bool wide = cdiv64(K1, kSlab) < 8 || u0 + u1 <= num_sms() / 2;
  if (int st = wide ? launch_pairs<8, 2>(m, p, u0, u1, s) : launch_pairs<4, 2>(m, p, u0, u1, s)) return st;
  return split > 1 ? launch_sum(o0, split, ws, s) : APA_OK;
}

// y = x W^T for up to 16 rows that the product casts itself.
int small_linear(const void* x, int x_dt, int64_t ld_x, const Operand& W, int64_t K, const OutArgs& o, cudaStream_t s) {
  const BlockPlan p = block_plan(o.M, o.N, K, o.vec && ((int64_t)o.N * elem_bytes(o.out_dt)) % 16 == 0);
  const RowArgs rows{x, ld_x, x_dt, vec16(x, ld_x, elem_bytes(x_dt)) ? 1 : 0, K};
  return launch_split<16, true>(W, Operand{nullptr, 0, nullptr, o.M}, K, o, true, p.split, s, rows);
}

}  // namespace blk
}  // namespace apa

namespace {

int gemm_dims(int64_t M, int64_t N, int64_t K) {
  if (M <= 0 || N <= 0 || K <= 0) return APA_ERR_INVALID;
  const int64_t top = (1ll << 31) - 256;
  return M > top || N > top || K > top ? APA_ERR_INVALID : APA_OK;
}

}  // namespace

extern "C" int apa_block_gemm_workspace(int64_t M, int64_t N, int64_t K, int out_dtype, int plan, int64_t* bytes_out) {
  using namespace apa::blk;
  if (!bytes_out) return APA_ERR_INVALID;
  if (int st = gemm_dims(M, N, K)) return st;
  if (elem_bytes(out_dtype) == 0) return APA_ERR_UNSUPPORTED;
  BlockPlan p{};
  if (plan != APA_BLOCK_AUTO) {
    if (int st = force_plan(plan, M, N, K, &p)) return st;
  } else {
    p = block_plan(M, N, K, (N * elem_bytes(out_dtype)) % 16 == 0);
  }
  *bytes_out = p.kind == 1 ? split_bytes(M, N, p.split) : 0;
  return APA_OK;
}

extern "C" int apa_block_gemm(const void* a, int64_t lda, const void* a_scales, const void* b, int64_t ldb,
                              const void* b_scales, const void* bias, int bias_dtype, void* out, int out_dtype,
                              int64_t ldo, int64_t M, int64_t N, int64_t K, int accumulate, int plan, void* workspace,
                              int64_t workspace_bytes, void* stream) {
  using namespace apa::blk;
  if (int st = gemm_dims(M, N, K)) return st;
  if (!a || !a_scales || !b || !b_scales || !out || lda < K || ldb < K || ldo < N) return APA_ERR_INVALID;
  const int es = elem_bytes(out_dtype);
  if (es == 0 || (bias && elem_bytes(bias_dtype) == 0)) return APA_ERR_UNSUPPORTED;
  if (accumulate && out_dtype != APA_DT_F32) return APA_ERR_UNSUPPORTED;
  if (!vec16(a, lda, 1) || !vec16(b, ldb, 1)) return APA_ERR_ALIGN;
  if (((reinterpret_cast<uintptr_t>(a_scales) | reinterpret_cast<uintptr_t>(b_scales) |
        reinterpret_cast<uintptr_t>(workspace)) & 15u) != 0)
    return APA_ERR_ALIGN;
  OutArgs o{out, ldo, out_dtype, bias, bias_dtype, accumulate ? 1 : 0, vec16(out, ldo, es) ? 1 : 0, (int)M, (int)N};
  const Operand A{a, lda, a_scales, M}, B{b, ldb, b_scales, N};
  BlockPlan p{};
  if (plan != APA_BLOCK_AUTO) {
    if (int st = force_plan(plan, M, N, K, &p)) return st;
  } else {
    p = block_plan(M, N, K, o.vec && (N * es) % 16 == 0);
  }
  if (p.kind == 1 && p.split > 1 && (!workspace || workspace_bytes < split_bytes(M, N, p.split))) {
    if (plan != APA_BLOCK_AUTO) return APA_ERR_INVALID;
    p.split = 1;      // without room for the slices: one unit per tile
  }
  return block_gemm(A, B, K, o, p, workspace, static_cast<cudaStream_t>(stream));
}
