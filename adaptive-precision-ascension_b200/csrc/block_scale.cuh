// E4M3 blocks with power-of-two scales: what the cast, the norm and the GEMM
// share.
//
// A block tensor holds the E4M3 codes of a [rows, K] matrix and one 8-bit
// exponent per row and 128 columns (OCP E8M0: byte b stands for 2^(b-127)).
// The value of an element is code * 2^(b-127). A scale is the smallest power
// of two s with max|block| <= 448 s, so no finite value saturates and
// multiplying by 1/s is exact (but for results below E4M3's subnormals).
// Powers of two, not arbitrary fp32 scales, because the tensor cores of
// sm_100a apply E8M0 scales themselves (tcgen05.mma kind::mxf8f6f4): the
// accumulator stays in tensor memory for the whole reduction, and dequantising
// adds no rounding.
//
// Scale storage: 32-bit words, one per row and four consecutive 128-column
// blocks (byte j of the word = block 4 kg + j), in the order tcgen05.cp and
// the MMA take: for each group kg of four blocks, rows in groups of 128, and
// inside a group row r at word (r % 32) * 4 + r / 32. rows_pad = rows rounded
// up to 128. So 128 rows x 512 columns have their scales in 512 contiguous
// bytes.
#pragma once

#include "apa_common.cuh"

namespace apa {
namespace blk {

constexpr int kBlock = 128;       // elements per scale along the reduction
constexpr int kGroupRows = 128;   // rows per scale chunk

__host__ __device__ __forceinline__ int64_t rows_padded(int64_t rows) {
  return (rows + kGroupRows - 1) / kGroupRows * kGroupRows;
}

// byte offset of the scale of (row, 128-column block kb)
__device__ __forceinline__ int64_t scale_offset(int64_t rows_pad, int64_t row, int64_t kb) {
  return ((kb >> 2) * rows_pad + (row & ~127ll) + (row & 31) * 4 + ((row >> 5) & 3)) * 4 + (kb & 3);
}

// Exponent byte of a block from the fp32 bits of its largest finite
// magnitude. amax = m 2^e (1 <= m < 2) and 448 = 1.75 2^8, so the smallest
// power of two is 2^(e-8) when m <= 1.75, else 2^(e-7). An empty (all zero)
// block gets 1. Exponents below 2^-126 are raised to it, so that both the
// scale and its reciprocal are normal fp32 numbers.
__device__ __forceinline__ uint32_t scale_byte(uint32_t amax_bits) {
  if (amax_bits == 0u) return 127u;
  const int b = (int)(amax_bits >> 23) - 8 + ((amax_bits & 0x7FFFFFu) > 0x600000u ? 1 : 0);
  return (uint32_t)max(b, 1);
}

// 1 / 2^(b-127); b in 1..247 here, so the result is normal and exact
__device__ __forceinline__ float inv_scale(uint32_t b) { return __uint_as_float((254u - b) << 23); }

// 2^(b-127) for any byte but 255: byte 0 is the subnormal 2^-127
__device__ __forceinline__ float scale_value(uint32_t b) {
  return __uint_as_float(b == 0u ? 0x00400000u : b << 23);
}

// m = max(m, |a|, |b|). NaN operands are skipped, so a maximum that starts at 0
// is a number; an infinity shows in it.
__device__ __forceinline__ float max_abs(float a, float b, float m) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(fabsf(a)), "f"(fabsf(b)), "f"(m));
  return r;
}

__device__ __forceinline__ bool is_inf(float a) { return __float_as_uint(a) == 0x7F800000u; }

// Infinities become NaN: E4M3 has no infinity, and the scale comes from the
// finite values. After this the saturating conversion gives the right codes:
// finite values are at most 448 in magnitude after scaling, where it rounds to
// nearest even, and it maps NaN to NaN.
__device__ __forceinline__ float inf_to_nan(float v) {
  return is_inf(fabsf(v)) ? __uint_as_float(0x7FC00000u) : v;
}

// Two products (or sums) per instruction, each rounded as the scalar one is.
__device__ __forceinline__ void mul2(float a0, float a1, float b0, float b1, float& d0, float& d1) {
  asm("{\n\t.reg .b64 a, b, d;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\t"
      "mul.rn.f32x2 d, a, b;\n\tmov.b64 {%0, %1}, d;\n\t}"
      : "=f"(d0), "=f"(d1)
      : "f"(a0), "f"(a1), "f"(b0), "f"(b1));
}
__device__ __forceinline__ void fma2(float a0, float a1, float b0, float b1, float c0, float c1, float& d0, float& d1) {
  asm("{\n\t.reg .b64 a, b, c, d;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tmov.b64 c, {%6, %7};\n\t"
      "fma.rn.f32x2 d, a, b, c;\n\tmov.b64 {%0, %1}, d;\n\t}"
      : "=f"(d0), "=f"(d1)
      : "f"(a0), "f"(a1), "f"(b0), "f"(b1), "f"(c0), "f"(c1));
}

// r * rstd * g with one rounding: the product r g is split into its rounded
// value and the exact remainder, and the last product is a fused one. A value
// next to a border of the E4M3 grid then lands on the side the exact product
// is on unless rstd's own rounding moves it.
__device__ __forceinline__ void normed8(float (&v)[8], float rstd, const float (&g)[8]) {
#pragma unroll
  for (int j = 0; j < 8; j += 2) {
    float t0, t1, e0, e1;
    mul2(v[j], v[j + 1], g[j], g[j + 1], t0, t1);
    fma2(v[j], v[j + 1], g[j], g[j + 1], -t0, -t1, e0, e1);
    mul2(e0, e1, rstd, rstd, e0, e1);
    fma2(t0, t1, rstd, rstd, e0, e1, v[j], v[j + 1]);
  }
}

template <int DT>
__device__ __forceinline__ float to_f32(const void* p, int64_t i) {
  if constexpr (DT == APA_DT_F32) return static_cast<const float*>(p)[i];
  else if constexpr (DT == APA_DT_F16) return f16_to_f32(static_cast<const uint16_t*>(p)[i]);
  else return bf16_to_f32(static_cast<const uint16_t*>(p)[i]);
}

__device__ __forceinline__ float to_f32(const void* p, int dt, int64_t i) {
  if (dt == APA_DT_F32) return to_f32<APA_DT_F32>(p, i);
  if (dt == APA_DT_F16) return to_f32<APA_DT_F16>(p, i);
  return to_f32<APA_DT_BF16>(p, i);
}

template <int DT>
__device__ __forceinline__ void from_f32(void* p, int64_t i, float v) {
  if constexpr (DT == APA_DT_F32) static_cast<float*>(p)[i] = v;
  else if constexpr (DT == APA_DT_F16) static_cast<uint16_t*>(p)[i] = f16_from_f32(v);
  else static_cast<uint16_t*>(p)[i] = bf16_from_f32(v);
}

__device__ __forceinline__ void from_f32(void* p, int dt, int64_t i, float v) {
  if (dt == APA_DT_F32) from_f32<APA_DT_F32>(p, i, v);
  else if (dt == APA_DT_F16) from_f32<APA_DT_F16>(p, i, v);
  else from_f32<APA_DT_BF16>(p, i, v);
}

__device__ __forceinline__ uint32_t bf16x2(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}

// Eight 16-bit elements -> fp32.
template <int DT>
__device__ __forceinline__ void unpack8(const uint4& a, float (&v)[8]) {
  const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    if constexpr (DT == APA_DT_BF16) {
      v[2 * j] = __uint_as_float(w[j] << 16);
      v[2 * j + 1] = __uint_as_float(w[j] & 0xFFFF0000u);
    } else {
      v[2 * j] = f16lo_to_f32(w[j]);
      v[2 * j + 1] = f16hi_to_f32(w[j]);
    }
  }
}

// Eight consecutive elements starting at i as fp32; n of them exist (the rest
// read as 0). vec: i is 16-byte aligned and all eight exist.
template <int DT>
__device__ __forceinline__ void load8(const void* p, int64_t i, int n, bool vec, float (&v)[8]) {
  if (vec) {
    if constexpr (DT == APA_DT_F32) {
      const float4 a = *reinterpret_cast<const float4*>(static_cast<const float*>(p) + i);
      const float4 b = *reinterpret_cast<const float4*>(static_cast<const float*>(p) + i + 4);
      v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
      v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
    } else {
      unpack8<DT>(*reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(p) + i), v);
    }
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = j < n ? to_f32<DT>(p, i + j) : 0.0f;
  }
}

// The same for an element type known at run time.
__device__ __forceinline__ void load8(const void* p, int dt, int64_t i, int n, bool vec, float (&v)[8]) {
  if (dt == APA_DT_F32) load8<APA_DT_F32>(p, i, n, vec, v);
  else if (dt == APA_DT_F16) load8<APA_DT_F16>(p, i, n, vec, v);
  else load8<APA_DT_BF16>(p, i, n, vec, v);
}

// Eight values times s -> eight codes (inf_to_nan first where there may be one).
__device__ __forceinline__ uint2 codes8(const float (&v)[8], float s) {
  float a[8];
#pragma unroll
  for (int j = 0; j < 8; j += 2) mul2(v[j], v[j + 1], s, s, a[j], a[j + 1]);
  return make_uint2(e4m3x2_sat(a[0], a[1]) | (e4m3x2_sat(a[2], a[3]) << 16),
                    e4m3x2_sat(a[4], a[5]) | (e4m3x2_sat(a[6], a[7]) << 16));
}

// Eight fp32 values -> eight 16-bit elements.
template <int DT>
__device__ __forceinline__ uint4 pack8(const float (&v)[8]) {
  uint32_t w[4];
#pragma unroll
  for (int j = 0; j < 4; ++j)
    w[j] = DT == APA_DT_BF16 ? bf16x2(v[2 * j], v[2 * j + 1]) : f16x2_from_f32(v[2 * j], v[2 * j + 1]);
  return make_uint4(w[0], w[1], w[2], w[3]);
}

template <int DT>
__device__ __forceinline__ void store8(void* p, int64_t i, int n, bool vec, const float (&v)[8]) {
  if (vec) {
    if constexpr (DT == APA_DT_F32) {
      float4* d = reinterpret_cast<float4*>(static_cast<float*>(p) + i);
      d[0] = make_float4(v[0], v[1], v[2], v[3]);
      d[1] = make_float4(v[4], v[5], v[6], v[7]);
    } else {
      *reinterpret_cast<uint4*>(static_cast<uint16_t*>(p) + i) = pack8<DT>(v);
    }
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (j < n) from_f32<DT>(p, i + j, v[j]);
  }
}

// Eight codes at 8-byte aligned d; n of them exist.
__device__ __forceinline__ void store_codes8(uint8_t* d, uint2 w, int n) {
  if (n >= 8) {
    *reinterpret_cast<uint2*>(d) = w;
  } else {
    const uint64_t b = ((uint64_t)w.y << 32) | w.x;
    for (int j = 0; j < n; ++j) d[j] = (uint8_t)(b >> (8 * j));
  }
}

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

// Raises a kernel's dynamic shared memory limit, which is a property of the
// kernel on a device: `done` holds a bit per device.
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

inline int elem_bytes(int dt) { return dt == APA_DT_F32 ? 4 : dt == APA_DT_F16 || dt == APA_DT_BF16 ? 2 : 0; }

inline bool vec16(const void* p, int64_t ld, int es) {
  return (reinterpret_cast<uintptr_t>(p) & 15u) == 0 && ((ld * es) & 15) == 0;
}

}  // namespace blk
}  // namespace apa
