// Casts between ordinary matrices and block tensors (E4M3 codes with one
// power-of-two scale per 128 elements; block_scale.cuh has the format).
//
//   rows form   q[r, c]   = RN_e4m3(x[r, c] / s[r, c / 128])
//   cols form   q_t[c, r] = RN_e4m3(x[r, c] / s_t[c, r / 128])
//   square      one scale per 128 x 128 for both forms (weights: the forward
//               and the input gradient then read the same values)
//
// The cols form is the K-major operand of a product that reduces over the
// rows (a weight gradient reduces over the tokens), so its scales run along
// the rows; it is not the rows form transposed. Optionally the source is
// x[r, c] * row_mul[r] * col_mul[c] (the norm's output recomputed from the
// residual stream), and the column sums of the source come along (the bias
// gradient), per 128 rows.
//
// Bound by HBM: every element is read once and written once per form. One
// 128 x 128 tile per CTA of 256 threads; a thread holds an 8 x 8 piece in
// registers, so both forms and all maxima come from one read.
#include "block_scale.cuh"

namespace apa {
namespace blk {

struct CastArgs {
  const void* src; int64_t rows, cols, ld_src;
  const float* row_mul; const void* col_mul; int col_mul_dt;
  uint8_t* dst; int64_t ld_dst; uint8_t* sc;
  uint8_t* dst_t; int64_t ld_dst_t; uint8_t* sc_t;
  float* colsum;
  int vec_src;
  int64_t tiles_c;
};

constexpr int kCastThreads = 256;

template <int SRC, bool SQUARE>
__global__ void __launch_bounds__(kCastThreads, 2) block_cast_kernel(CastArgs p) {
  __shared__ __align__(16) uint8_t s_t[128 * 128];
  __shared__ uint32_t s_max[8][128];
  __shared__ float s_sum[8][128];
  __shared__ uint32_t s_byte[128];
  pdl_launch_dependents();
  pdl_wait();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int g = lane & 15;                              // columns 8 g .. 8 g + 7
  const int lr0 = warp * 16 + (lane >> 4) * 8;          // rows lr0 .. lr0 + 7
  const int64_t tile_r = blockIdx.x / p.tiles_c, tile_c = blockIdx.x % p.tiles_c;
  const int64_t row0 = tile_r * 128, col0 = tile_c * 128;
  const int64_t c0 = col0 + 8 * g;
  const int nc = (int)max((int64_t)0, min((int64_t)8, p.cols - c0));
  const bool vec = p.vec_src && nc == 8;

  float v[8][8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int64_t r = row0 + lr0 + i;
    const int n = r < p.rows ? nc : 0;
    load8<SRC>(p.src, r * p.ld_src + c0, n, vec && n == 8, v[i]);
  }
  if (p.row_mul != nullptr) {
    float gm[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) gm[j] = j < nc ? to_f32(p.col_mul, p.col_mul_dt, c0 + j) : 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int64_t r = row0 + lr0 + i;
      const float rs = r < p.rows ? p.row_mul[r] : 0.0f;
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (r < p.rows && j < nc) v[i][j] = normed(v[i][j], rs, gm[j]);
    }
  }
  if (p.colsum != nullptr) {
    // column sums in a fixed order: eight rows per thread, two half warps,
    // eight warps
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      float t = v[0][j];
#pragma unroll
      for (int i = 1; i < 8; ++i) t += v[i][j];
      t += __shfl_xor_sync(0xFFFFFFFFu, t, 16);
      if (lane < 16) s_sum[warp][8 * g + j] = t;
    }
  }

  uint32_t rm[8], cm[8], all = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) rm[i] = 0;
#pragma unroll
  for (int j = 0; j < 8; ++j) cm[j] = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i)
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const uint32_t a = mag_bits(v[i][j]);
      rm[i] = max(rm[i], a);
      cm[j] = max(cm[j], a);
    }
#pragma unroll
  for (int i = 0; i < 8; ++i) all = max(all, rm[i]);
  const bool odd = bits_nonfinite(all);
  if (odd) {
    // rare: scales come from the finite values alone
    all = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) rm[i] = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) cm[j] = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i)
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const uint32_t a = finite_mag(v[i][j]);
        rm[i] = max(rm[i], a);
        cm[j] = max(cm[j], a);
        all = max(all, a);
      }
  }

  const int64_t kb_c = tile_c, kb_r = tile_r;
  const int64_t rows_pad = rows_padded(p.rows), cols_pad = rows_padded(p.cols);
  uint32_t byte_all = 0;
  if constexpr (SQUARE) {
    const uint32_t w = warp_max_u32(all);
    if (lane == 0) s_max[0][warp] = w;
    __syncthreads();
    uint32_t m = 0;
#pragma unroll
    for (int k = 0; k < 8; ++k) m = max(m, s_max[0][k]);
    byte_all = scale_byte(m);
  }

  if (p.dst != nullptr) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      uint32_t b;
      if constexpr (SQUARE) {
        b = byte_all;
      } else {
        uint32_t m = rm[i];
#pragma unroll
        for (int o = 8; o > 0; o >>= 1) m = max(m, __shfl_xor_sync(0xFFFFFFFFu, m, o));
        b = scale_byte(m);
      }
      const float is = inv_scale(b);
      const int64_t r = row0 + lr0 + i;
      // rows past the end, up to the next multiple of 128, have a scale too
      if (g == 0) p.sc[scale_offset(rows_pad, r, kb_c)] = (uint8_t)b;
      if (r < p.rows && nc > 0) {
        uint2 w;
        w.x = codes2(v[i][0] * is, v[i][1] * is, odd) | (codes2(v[i][2] * is, v[i][3] * is, odd) << 16);
        w.y = codes2(v[i][4] * is, v[i][5] * is, odd) | (codes2(v[i][6] * is, v[i][7] * is, odd) << 16);
        store_codes8(p.dst + r * p.ld_dst + c0, w, nc);
      }
    }
  }

  if (p.dst_t != nullptr || p.colsum != nullptr) {
    if (!SQUARE && p.dst_t != nullptr) {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const uint32_t m = max(cm[j], __shfl_xor_sync(0xFFFFFFFFu, cm[j], 16));
        if (lane < 16) s_max[warp][8 * g + j] = m;
      }
    }
    __syncthreads();
    if (threadIdx.x < 128) {
      const int c = threadIdx.x;
      if (p.dst_t != nullptr) {
        uint32_t b = byte_all;
        if constexpr (!SQUARE) {
          uint32_t m = 0;
#pragma unroll
          for (int k = 0; k < 8; ++k) m = max(m, s_max[k][c]);
          b = scale_byte(m);
        }
        s_byte[c] = b;
        p.sc_t[scale_offset(cols_pad, col0 + c, kb_r)] = (uint8_t)b;
      }
      if (p.colsum != nullptr && col0 + c < p.cols) {
        float t = s_sum[0][c];
#pragma unroll
        for (int k = 1; k < 8; ++k) t += s_sum[k][c];
        p.colsum[tile_r * p.cols + col0 + c] = t;
      }
    }
    if (p.dst_t == nullptr) return;
    __syncthreads();
    // s_t[c][r]: row c in 16 chunks of 8 bytes, chunk k at k ^ (c / 8), so that
    // the sixteen lanes of a half warp (one chunk, sixteen column groups)
    // write to distinct banks
    const int chunk = lr0 >> 3;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float is = inv_scale(s_byte[8 * g + j]);
      uint2 w;
      w.x = codes2(v[0][j] * is, v[1][j] * is, odd) | (codes2(v[2][j] * is, v[3][j] * is, odd) << 16);
      w.y = codes2(v[4][j] * is, v[5][j] * is, odd) | (codes2(v[6][j] * is, v[7][j] * is, odd) << 16);
      *reinterpret_cast<uint2*>(s_t + (8 * g + j) * 128 + ((chunk ^ g) << 3)) = w;
    }
    __syncthreads();
    // eight threads per column, 16 bytes each; odd columns read their two
    // chunks in the other order, which keeps the half warp's banks distinct
    const int k2 = threadIdx.x & 7;
#pragma unroll
    for (int it = 0; it < 4; ++it) {
      const int c = it * 32 + (threadIdx.x >> 3);
      const int64_t gc = col0 + c, gr = row0 + 16 * k2;
      const int sw = c >> 3, first = c & 1;
      const uint8_t* base = s_t + c * 128;
      const uint2 a = *reinterpret_cast<const uint2*>(base + (((2 * k2 + first) ^ sw) << 3));
      const uint2 b = *reinterpret_cast<const uint2*>(base + (((2 * k2 + (first ^ 1)) ^ sw) << 3));
      const uint2 lo = first ? b : a, hi = first ? a : b;
      if (gc < p.cols && gr < p.rows) {
        uint8_t* d = p.dst_t + gc * p.ld_dst_t + gr;
        const int64_t n = p.rows - gr;
        if (n >= 16) {
          *reinterpret_cast<uint4*>(d) = make_uint4(lo.x, lo.y, hi.x, hi.y);
        } else {
          store_codes8(d, lo, (int)min(n, (int64_t)8));
          if (n > 8) store_codes8(d + 8, hi, (int)n - 8);
        }
      }
    }
  }
}

struct DequantArgs {
  const uint8_t* src; int64_t ld; const uint8_t* sc;
  int64_t rows, cols; void* dst; int64_t ld_dst;
  int vec_dst;
  int64_t chunks;   // 16-element chunks per row
};

// One thread per 16 codes (one 16-byte load).
template <int DST>
__global__ void __launch_bounds__(256) block_dequant_kernel(DequantArgs p) {
  pdl_launch_dependents();
  pdl_wait();
  const int64_t total = p.rows * p.chunks;
  const int64_t rows_pad = rows_padded(p.rows);
  for (int64_t e = (int64_t)blockIdx.x * 256 + threadIdx.x; e < total; e += (int64_t)gridDim.x * 256) {
    const int64_t r = e / p.chunks, c0 = (e - r * p.chunks) * 16;
    const uint4 q = *reinterpret_cast<const uint4*>(p.src + r * p.ld + c0);   // rows are padded to 16 codes
    const float s = scale_value(p.sc[scale_offset(rows_pad, r, c0 >> 7)]);
    const uint32_t w[4] = {q.x, q.y, q.z, q.w};
    const int n = (int)min((int64_t)16, p.cols - c0);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      float v[8];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const uint32_t two = (w[2 * h + (k >> 1)] >> (16 * (k & 1))) & 0xFFFFu;
        const uint32_t f = f16x2_from_e4m3x2(two);
        v[2 * k] = f16lo_to_f32(f) * s;
        v[2 * k + 1] = f16hi_to_f32(f) * s;
      }
      const int nn = min(8, n - 8 * h);
      if (nn > 0) store8<DST>(p.dst, r * p.ld_dst + c0 + 8 * h, nn, p.vec_dst && nn == 8, v);
    }
  }
}

// Column sums of [parts, cols] fp32 partials in a fixed order, rounded once to
// the output's type. 32 columns x 32 warps per CTA, warp w takes rows w, w+32, ..
__global__ void __launch_bounds__(1024) block_colsum_kernel(const float* part, int64_t parts, int64_t cols, void* out,
                                                            int out_dt) {
  pdl_launch_dependents();
  pdl_wait();
  __shared__ float s[32][33];
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  const int64_t c = (int64_t)blockIdx.x * 32 + lane;
  float t = 0.0f;
  if (c < cols) {
    int64_t r = w;
    for (; r + 7 * 32 < parts; r += 8 * 32) {
      float x[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) x[k] = part[(r + 32 * k) * cols + c];
#pragma unroll
      for (int k = 0; k < 8; ++k) t += x[k];
    }
    for (; r < parts; r += 32) t += part[r * cols + c];
  }
  s[w][lane] = t;
  __syncthreads();
  // column `w` of the CTA is summed by warp w: lanes hold its 32 partials
  float u = s[lane][w];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) u += __shfl_xor_sync(0xFFFFFFFFu, u, o);
  const int64_t oc = (int64_t)blockIdx.x * 32 + w;
  if (lane == 0 && oc < cols) from_f32(out, out_dt, oc, u);
}

int launch_colsum(const float* part, int64_t parts, int64_t cols, void* out, int out_dt, cudaStream_t s) {
  const int64_t grid = (cols + 31) / 32;
  return launch_kernel(block_colsum_kernel, dim3((unsigned)grid), dim3(1024), 0, s, 1, part, parts, cols, out,
                       out_dt) == cudaSuccess ? APA_OK : APA_ERR_CUDA;
}

}  // namespace blk
}  // namespace apa

extern "C" int apa_block_cast(const void* src, int src_dtype, int64_t rows, int64_t cols, int64_t ld_src,
                              const float* row_mul, const void* col_mul, int col_mul_dtype, int square, void* dst,
                              int64_t ld_dst, void* scales, void* dst_t, int64_t ld_dst_t, void* scales_t,
                              float* colsum_partial, void* stream) {
  using namespace apa::blk;
  if (!src || rows <= 0 || cols <= 0 || ld_src < cols) return APA_ERR_INVALID;
  if (rows > (1ll << 31) - 256 || cols > (1ll << 31) - 256) return APA_ERR_INVALID;
  if ((dst == nullptr) != (scales == nullptr) || (dst_t == nullptr) != (scales_t == nullptr)) return APA_ERR_INVALID;
  if (!dst && !dst_t) return APA_ERR_INVALID;
  if ((dst && ld_dst < cols) || (dst_t && ld_dst_t < rows)) return APA_ERR_INVALID;
  if ((row_mul == nullptr) != (col_mul == nullptr)) return APA_ERR_INVALID;
  const int es = elem_bytes(src_dtype);
  if (es == 0 || (col_mul && elem_bytes(col_mul_dtype) == 0)) return APA_ERR_UNSUPPORTED;
  if (dst && !vec16(dst, ld_dst, 1)) return APA_ERR_ALIGN;
  if (dst_t && !vec16(dst_t, ld_dst_t, 1)) return APA_ERR_ALIGN;
  const int64_t tr = (rows + 127) / 128, tc = (cols + 127) / 128;
  if (tr * tc > (1ll << 31) - 1) return APA_ERR_INVALID;
  CastArgs a{src, rows, cols, ld_src, row_mul, col_mul, col_mul_dtype, static_cast<uint8_t*>(dst), ld_dst,
             static_cast<uint8_t*>(scales), static_cast<uint8_t*>(dst_t), ld_dst_t, static_cast<uint8_t*>(scales_t),
             colsum_partial, vec16(src, ld_src, es) ? 1 : 0, tc};
  void (*k)(CastArgs);
  if (src_dtype == APA_DT_F32) k = square ? block_cast_kernel<APA_DT_F32, true> : block_cast_kernel<APA_DT_F32, false>;
  else if (src_dtype == APA_DT_F16) k = square ? block_cast_kernel<APA_DT_F16, true> : block_cast_kernel<APA_DT_F16, false>;
  else k = square ? block_cast_kernel<APA_DT_BF16, true> : block_cast_kernel<APA_DT_BF16, false>;
  return apa::launch_kernel(k, dim3((unsigned)(tr * tc)), dim3(kCastThreads), 0, static_cast<cudaStream_t>(stream), 1,
                            a) == cudaSuccess ? APA_OK : APA_ERR_CUDA;
}

extern "C" int apa_block_dequant(const void* src, int64_t ld, const void* scales, int64_t rows, int64_t cols, void* dst,
                                 int dst_dtype, int64_t ld_dst, void* stream) {
  using namespace apa::blk;
  if (!src || !scales || !dst || rows <= 0 || cols <= 0 || ld < cols || ld_dst < cols) return APA_ERR_INVALID;
  if (rows > (1ll << 31) - 256 || cols > (1ll << 31) - 256) return APA_ERR_INVALID;
  const int es = elem_bytes(dst_dtype);
  if (es == 0) return APA_ERR_UNSUPPORTED;
  if (!vec16(src, ld, 1)) return APA_ERR_ALIGN;
  DequantArgs a{static_cast<const uint8_t*>(src), ld, static_cast<const uint8_t*>(scales), rows, cols, dst, ld_dst,
                vec16(dst, ld_dst, es) ? 1 : 0, (cols + 15) / 16};
  const int64_t grid = std::min<int64_t>((rows * a.chunks + 255) / 256, (int64_t)apa::num_sms() * 16);
  void (*k)(DequantArgs) = dst_dtype == APA_DT_F32 ? block_dequant_kernel<APA_DT_F32>
                           : dst_dtype == APA_DT_F16 ? block_dequant_kernel<APA_DT_F16>
                                                     : block_dequant_kernel<APA_DT_BF16>;
  return apa::launch_kernel(k, dim3((unsigned)grid), dim3(256), 0, static_cast<cudaStream_t>(stream), 1, a) ==
                 cudaSuccess ? APA_OK : APA_ERR_CUDA;
}

extern "C" int apa_block_colsum(const float* partial, int64_t parts, int64_t cols, void* out, int out_dtype,
                                void* stream) {
  using namespace apa::blk;
  if (!partial || !out || parts <= 0 || cols <= 0 || cols > (1ll << 31) - 256) return APA_ERR_INVALID;
  if (elem_bytes(out_dtype) == 0) return APA_ERR_UNSUPPORTED;
  return launch_colsum(partial, parts, cols, out, out_dtype, static_cast<cudaStream_t>(stream));
}
