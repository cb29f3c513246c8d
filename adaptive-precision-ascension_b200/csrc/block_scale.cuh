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

// max of magnitudes (fp32 bits) that skips NaN and Inf. Kernels take the plain
// maximum first (fmaxf skips NaN) and come here only when that is infinite.
__device__ __forceinline__ float finite_mag(float v) {
  const float a = fabsf(v);
  return a < __uint_as_float(0x7F800000u) ? a : 0.0f;
}

__device__ __forceinline__ bool is_inf(float a) { return __float_as_uint(a) == 0x7F800000u; }

// Scaled values -> codes. Finite values are at most 448 in magnitude after
// scaling, where the saturating conversion rounds to nearest even like the
// exact one, and it maps NaN to NaN. Only an infinity needs the exact rule (NaN;
// E4M3 has no infinity): odd says that the thread holds one.

// r * rstd * g with one rounding: the product r g is split into its rounded
// value and the exact remainder, and the last product is a fused one. A value
// next to a border of the E4M3 grid then lands on the side the exact product
// is on unless rstd's own rounding moves it.
__device__ __forceinline__ float normed(float r, float rstd, float g) {
  const float t = __fmul_rn(r, g);
  const float e = __fmaf_rn(r, g, -t);
  return __fmaf_rn(t, rstd, __fmul_rn(e, rstd));
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

template <int DT>
__device__ __forceinline__ float round_to(float v) {
  if constexpr (DT == APA_DT_F16) return f16_to_f32(f16_from_f32(v));
  else if constexpr (DT == APA_DT_BF16) return bf16_to_f32(bf16_from_f32(v));
  else return v;
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

// Eight scaled values -> eight codes.
__device__ __forceinline__ uint2 codes8(const float (&v)[8], float s, bool odd) {
  uint2 w;
  if (!odd) {
    w.x = e4m3x2_sat(v[0] * s, v[1] * s) | (e4m3x2_sat(v[2] * s, v[3] * s) << 16);
    w.y = e4m3x2_sat(v[4] * s, v[5] * s) | (e4m3x2_sat(v[6] * s, v[7] * s) << 16);
  } else {
    w.x = e4m3x2_exact(v[0] * s, v[1] * s) | (e4m3x2_exact(v[2] * s, v[3] * s) << 16);
    w.y = e4m3x2_exact(v[4] * s, v[5] * s) | (e4m3x2_exact(v[6] * s, v[7] * s) << 16);
  }
  return w;
}

template <int DT>
__device__ __forceinline__ void store8(void* p, int64_t i, int n, bool vec, const float (&v)[8]) {
  if (vec) {
    if constexpr (DT == APA_DT_F32) {
      float4* d = reinterpret_cast<float4*>(static_cast<float*>(p) + i);
      d[0] = make_float4(v[0], v[1], v[2], v[3]);
      d[1] = make_float4(v[4], v[5], v[6], v[7]);
    } else {
      uint32_t w[4];
#pragma unroll
      for (int j = 0; j < 4; ++j)
        w[j] = DT == APA_DT_BF16 ? bf16x2(v[2 * j], v[2 * j + 1]) : f16x2_from_f32(v[2 * j], v[2 * j + 1]);
      *reinterpret_cast<uint4*>(static_cast<uint16_t*>(p) + i) = make_uint4(w[0], w[1], w[2], w[3]);
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

inline int elem_bytes(int dt) { return dt == APA_DT_F32 ? 4 : dt == APA_DT_F16 || dt == APA_DT_BF16 ? 2 : 0; }

inline bool vec16(const void* p, int64_t ld, int es) {
  return (reinterpret_cast<uintptr_t>(p) & 15u) == 0 && ((ld * es) & 15) == 0;
}

}  // namespace blk
}  // namespace apa
