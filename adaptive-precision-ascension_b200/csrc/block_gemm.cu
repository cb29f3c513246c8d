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
// split_kernel  one 128 x BN tile (BN 16 to 128) on one CTA, the reduction
//   split over the CTAs of a cluster, whose partial tiles meet in distributed
//   shared memory and are added in rank order. For problems with too few
//   256 x 256 tiles to fill the GPU: with few tokens (swapped: the 128 side
//   holds the weight's rows) it is bound by reading the weight, and S CTAs per
//   tile keep every SM's loads in flight; for a small weight gradient over
//   many tokens the split is what fills the SMs. No workspace, no atomics: the
//   result does not depend on timing.
#include <cuda.h>
#include <mutex>
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

// C consecutive accumulator columns of one row. Not swapped: row m, columns
// n0 ..; swapped: weight row n of tokens m0 .. (neighbouring lanes hold
// neighbouring n, so every store instruction writes whole sectors).
template <int C>
__device__ __forceinline__ void put(const OutArgs& o, bool swap, int row, int col, float (&v)[C]) {
  if (swap) {
    const int n = row;
    if (n >= o.N) return;
    const float b = o.bias ? to_f32(o.bias, o.bias_dt, n) : 0.0f;
#pragma unroll
    for (int j = 0; j < C; ++j) {
      const int m = col + j;
      if (m < o.M) {
        const int64_t at = (int64_t)m * o.ldo + n;
        float x = v[j] + b;
        if (o.accumulate) x += static_cast<const float*>(o.out)[at];
        from_f32(o.out, o.out_dt, at, x);
      }
    }
    return;
  }
  const int m = row;
  if (m >= o.M || col >= o.N) return;
  const int64_t at = (int64_t)m * o.ldo + col;
  if (o.bias) {
#pragma unroll
    for (int j = 0; j < C; ++j)
      if (col + j < o.N) v[j] += to_f32(o.bias, o.bias_dt, col + j);
  }
  if (C % 8 == 0 && o.vec && col + C <= o.N) {
    if (o.out_dt == APA_DT_F32) {
      float4* d = reinterpret_cast<float4*>(static_cast<float*>(o.out) + at);
#pragma unroll
      for (int q = 0; q < C / 4; ++q) {
        float4 x = make_float4(v[4 * q], v[4 * q + 1], v[4 * q + 2], v[4 * q + 3]);
        if (o.accumulate) {
          const float4 y = d[q];
          x.x += y.x; x.y += y.y; x.z += y.z; x.w += y.w;
        }
        d[q] = x;
      }
    } else {
      uint4* d = reinterpret_cast<uint4*>(static_cast<uint16_t*>(o.out) + at);
      uint32_t w[C / 2];
#pragma unroll
      for (int j = 0; j < C / 2; ++j)
        w[j] = o.out_dt == APA_DT_BF16 ? bf16x2(v[2 * j], v[2 * j + 1]) : f16x2_from_f32(v[2 * j], v[2 * j + 1]);
#pragma unroll
      for (int q = 0; q < C / 8; ++q) d[q] = make_uint4(w[4 * q], w[4 * q + 1], w[4 * q + 2], w[4 * q + 3]);
    }
    return;
  }
#pragma unroll
  for (int j = 0; j < C; ++j) {
    if (col + j < o.N) {
      float x = v[j];
      if (o.accumulate) x += static_cast<const float*>(o.out)[at + j];
      from_f32(o.out, o.out_dt, at + j, x);
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
  // two CTAs per SM (one loads while the other finishes)
  static constexpr int kStages = BN == 128 ? 3 : BN == 64 ? 4 : 5;
  static constexpr int kTmemCols = BN == 128 ? 256 : BN == 64 ? 128 : BN == 32 ? 64 : 32;
  static constexpr int kSmemBytes = kStages * (kStageBytes + kScaleBytes) + 1024 + 256;
  static constexpr int kThreads = 192;
  static_assert(BN * BM * 4 <= kStages * kStageBytes, "the partial tile reuses the stages");
  static_assert(BN + 8 <= kTmemCols, "tensor memory");
  static_assert(2 * (kSmemBytes + 1024) <= 228 * 1024, "two CTAs per SM");
};

struct SplitArgs {
  int rows_a, rows_b;       // rows of the 128 side and of the BN side
  int tiles_b;
  int kb_count;             // 128-column slabs
  int split;                // CTAs per tile (cluster size)
  int swap;                 // the 128 side is D's N
  OutArgs o;
};

template <int BN>
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
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(done + 1);
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
        mbar_expect_tx(&full[stage], C::kStageBytes + (scales ? C::kScaleBytes : 0));
        tma_load_2d(smA + stage * C::kABytes, &tmA, kb * kSlab, a0, &full[stage]);
        tma_load_2d(smB + stage * C::kBBytes, &tmB, kb * kSlab, b0, &full[stage]);
        if (scales) {
          uint8_t* s = smS + stage * C::kScaleBytes;
          tma_load_2d(s, &tmSA, a0, kb >> 2, &full[stage]);
          tma_load_2d(s + 512, &tmSB, b0 & ~127, kb >> 2, &full[stage]);
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
      // rows b0 .. of a chunk of 128 start at scale column (b0 % 128) / 32
      const uint32_t sfb0 = sfb + (uint32_t)((b0 & 127) >> 5);
      for (int kb = kb0; kb < kb1; ++kb) {
        if (!mbar_wait(&full[stage], phase, kStatusTimeoutFull)) { ok = false; break; }
        fence_after();
        if (kb == kb0 || (kb & 3) == 0) {
          const uint32_t s = smem_u32(smS + stage * C::kScaleBytes);
          scale_copy<false>(sfa, s);
          scale_copy<false>(sfb, s + 512);
        }
        const uint32_t j = (uint32_t)(kb & 3);
        const uint32_t id = mx_idesc<BN, BM>() | (j << 4) | (j << 29);
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

  // epilogue: warps 2 .. 5 read the accumulator's lane quarter warp % 4
  const int q = warp & 3;
  bool ready = false;
  if (warp >= 2) {
    if (lane == 0) ready = mbar_wait(done, 0, kStatusTimeoutAcc);
    ready = __shfl_sync(0xFFFFFFFFu, ready ? 1 : 0, 0) != 0;
    fence_after();
  }
  const uint32_t lanes = tmem + ((uint32_t)(q * 32) << 16);
  const int row = a0 + q * 32 + lane;
  constexpr int kC = BN >= 32 ? 32 : 16;
  if (p.split == 1) {
    if (warp >= 2 && ready) {
#pragma unroll 1
      for (int c = 0; c < BN; c += kC) {
        if (b0 + c >= p.rows_b) break;
        uint32_t r[kC];
        if constexpr (kC == 32) gemm::tmem_ld32_nowait(lanes + c, r);
        else tmem_ld16(lanes + c, r);
        gemm::tmem_wait_ld();
        float v[kC];
#pragma unroll
        for (int j = 0; j < kC; ++j) v[j] = fu(r[j]);
        put<kC>(p.o, p.swap != 0, row, b0 + c, v);
      }
    }
  } else {
    // partial tiles, column major ([BN][128] fp32), over the operand stages:
    // every load has landed and every MMA has read it once `done` completes
    float* part = reinterpret_cast<float*>(smem);
    if (warp >= 2 && ready) {
#pragma unroll 1
      for (int c = 0; c < BN; c += kC) {
        uint32_t r[kC];
        if constexpr (kC == 32) gemm::tmem_ld32_nowait(lanes + c, r);
        else tmem_ld16(lanes + c, r);
        gemm::tmem_wait_ld();
#pragma unroll
        for (int j = 0; j < kC; ++j) part[(c + j) * BM + q * 32 + lane] = fu(r[j]);
      }
    }
    __syncwarp();
    gemm::cluster_sync();
    if (warp >= 2 && ready) {
      // this rank's columns (split <= 8), in groups that make 16-byte stores
      // where a rank has eight columns or more
      constexpr int kG = BN >= 64 ? 8 : 2;
      const int per = BN / p.split;
      for (int c = rank * per; c < (rank + 1) * per; c += kG) {
        if (b0 + c >= p.rows_b) break;
        float v[kG];
#pragma unroll
        for (int j = 0; j < kG; ++j) v[j] = 0.0f;
        for (int s = 0; s < p.split; ++s) {
          const uint32_t at = gemm::map_to_cta(part + c * BM + q * 32 + lane, (uint32_t)s);
#pragma unroll
          for (int j = 0; j < kG; ++j) {
            float x;
            asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(x) : "r"(at + (uint32_t)(j * BM * 4)));
            v[j] += x;
          }
        }
        put<kG>(p.o, p.swap != 0, row, b0 + c, v);
      }
    }
    __syncwarp();
    gemm::cluster_sync();   // no CTA leaves while another reads its partials
  }
  fence_before();
  __syncthreads();
  fence_after();
  if (warp == 1)
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"((uint32_t)C::kTmemCols)
                 : "memory");
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

struct Operand { const void* q; int64_t ld; const void* sc; int64_t rows; };

// The dynamic shared memory limit is a property of a kernel on a device.
template <class K>
int allow_smem(K kernel, int bytes, unsigned long long* done) {
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return APA_ERR_CUDA;
  const unsigned long long bit = 1ull << (dev & 63);
  if (__atomic_load_n(done, __ATOMIC_ACQUIRE) & bit) return APA_OK;
  if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) != cudaSuccess)
    return APA_ERR_CUDA;
  __atomic_fetch_or(done, bit, __ATOMIC_RELEASE);
  return APA_OK;
}

template <int BN>
int launch_split(const Operand& A, const Operand& B, int64_t K, const OutArgs& o, bool swap, int split,
                 cudaStream_t s) {
  using C = SplitCfg<BN>;
  static unsigned long long attr = 0;
  if (int st = allow_smem(split_kernel<BN>, C::kSmemBytes, &attr)) return st;
  const int64_t kb = (K + kSlab - 1) / kSlab;
  CUtensorMap ta, tb, tsa, tsb;
  if (int st = code_map(&ta, A.q, A.rows, K, A.ld, BM)) return st;
  if (int st = code_map(&tb, B.q, B.rows, K, B.ld, BN)) return st;
  if (int st = scale_map(&tsa, A.sc, A.rows, kb, 128)) return st;
  if (int st = scale_map(&tsb, B.sc, B.rows, kb, 128)) return st;
  SplitArgs p;
  p.rows_a = (int)A.rows; p.rows_b = (int)B.rows;
  p.tiles_b = (int)((B.rows + BN - 1) / BN);
  p.kb_count = (int)kb; p.split = split; p.swap = swap ? 1 : 0; p.o = o;
  const int64_t grid = (A.rows + BM - 1) / BM * p.tiles_b * split;
  if (grid > (1ll << 31) - 1) return APA_ERR_INVALID;
  return launch_kernel(split_kernel<BN>, dim3((unsigned)grid), dim3(C::kThreads), C::kSmemBytes, s, split, ta, tb, tsa,
                       tsb, p) == cudaSuccess ? APA_OK : APA_ERR_CUDA;
}

struct BlockPlan { int kind, bn, split, swap; };   // kind 0: split_kernel

int64_t cdiv64(int64_t a, int64_t b) { return (a + b - 1) / b; }

BlockPlan block_plan(int64_t M, int64_t N, int64_t K) {
  BlockPlan p{0, 128, 1, 0};
  const int64_t kb = cdiv64(K, kSlab);
  p.swap = M <= 128 && M < N;
  const int64_t small = p.swap ? M : N, big = p.swap ? N : M;
  p.bn = small <= 16 ? 16 : small <= 32 ? 32 : small <= 64 ? 64 : 128;
  const int64_t tiles = cdiv64(big, BM) * cdiv64(small, p.bn);
  while (p.split < 8 && tiles * p.split * 2 <= 2 * num_sms() && p.split * 2 * 2 <= kb) p.split *= 2;
  return p;
}

int block_gemm(const Operand& A, const Operand& B, int64_t K, const OutArgs& o, const BlockPlan& p, cudaStream_t s) {
  const Operand& x = p.swap ? B : A;
  const Operand& y = p.swap ? A : B;
  switch (p.bn) {
    case 16: return launch_split<16>(x, y, K, o, p.swap, p.split, s);
    case 32: return launch_split<32>(x, y, K, o, p.swap, p.split, s);
    case 64: return launch_split<64>(x, y, K, o, p.swap, p.split, s);
    default: return launch_split<128>(x, y, K, o, p.swap, p.split, s);
  }
}

}  // namespace blk
}  // namespace apa

extern "C" int apa_block_gemm(const void* a, int64_t lda, const void* a_scales, const void* b, int64_t ldb,
                              const void* b_scales, const void* bias, int bias_dtype, void* out, int out_dtype,
                              int64_t ldo, int64_t M, int64_t N, int64_t K, int accumulate, void* stream) {
  using namespace apa::blk;
  if (M <= 0 || N <= 0 || K <= 0) return APA_ERR_INVALID;
  if (M > (1ll << 31) - 256 || N > (1ll << 31) - 256 || K > (1ll << 31) - 256) return APA_ERR_INVALID;
  if (!a || !a_scales || !b || !b_scales || !out || lda < K || ldb < K || ldo < N) return APA_ERR_INVALID;
  const int es = elem_bytes(out_dtype);
  if (es == 0 || (bias && elem_bytes(bias_dtype) == 0)) return APA_ERR_UNSUPPORTED;
  if (accumulate && out_dtype != APA_DT_F32) return APA_ERR_UNSUPPORTED;
  if (!vec16(a, lda, 1) || !vec16(b, ldb, 1)) return APA_ERR_ALIGN;
  if (((reinterpret_cast<uintptr_t>(a_scales) | reinterpret_cast<uintptr_t>(b_scales)) & 15u) != 0) return APA_ERR_ALIGN;
  OutArgs o{out, ldo, out_dtype, bias, bias_dtype, accumulate ? 1 : 0, vec16(out, ldo, es) ? 1 : 0, (int)M, (int)N};
  const Operand A{a, lda, a_scales, M}, B{b, ldb, b_scales, N};
  const BlockPlan p = block_plan(M, N, K);
  return block_gemm(A, B, K, o, p, static_cast<cudaStream_t>(stream));
}
