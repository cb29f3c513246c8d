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
// Every element is read once and written once per form. fp32 sources run at
// HBM's rate. 16-bit ones reach no unit's limit (ALU pipe 57 %, issue slots
// 61 %): two CTAs fill the register file, 46 % of the warps, and each passes up
// to three barriers a tile, so what a tile waits for is not hidden. One
// 128 x 128 tile per CTA of 512 threads; a thread holds a 4 x 8 piece in
// registers, so both forms and all maxima come from one read, and 64 registers
// a thread leave room for two CTAs per SM. (8 x 8 pieces on 256 threads ran at
// a third of the speed; persistent CTAs with the next tile fetched ahead by
// cp.async gained nothing in bf16 and lost a third in fp32.)
//
// Measured on a B200, inputs in HBM, 8192 x 4096 (us, TB/s of what is read and
// written): bf16 rows form 20.5, 4.9; cols 23.9, 4.2; both 30.3, 4.4; fp32 rows
// 26.3, 6.4; both 34.2, 5.9. Dequantisation to bf16 19.4, 5.2.
#include "block_scale.cuh"

namespace apa {
namespace blk {

struct CastArgs {
  const void* src; int64_t rows, cols, ld_src;
  const float* row_mul; const void* col_mul; int col_mul_dt;
  uint8_t* dst; int64_t ld_dst; uint8_t* sc;
  uint8_t* dst_t; int64_t ld_dst_t; uint8_t* sc_t;
  float* colsum;
  int vec_src, vec_mul;
  int64_t tiles_c;
};

constexpr int kCastThreads = 512;

struct CastShared {
  uint32_t t[128 * 32];          // transposed codes, 128 bytes per column
  float max[16][128];            // column maxima per warp
  float sum[16][128];
  float inv[128];
};

// One 128 x 128 tile. NORM: the source is src * row_mul * col_mul. (Maxima of
// 16-bit sources on packed pairs, half the instructions, were no faster at two
// CTAs per SM.)
template <int SRC, bool SQUARE, bool NORM>
__device__ __forceinline__ void cast_tile(const CastArgs& p, int64_t tile, CastShared& sm) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int g = lane & 15, half = lane >> 4;            // columns 8 g .. 8 g + 7
  const int lr0 = warp * 8 + half * 4;                  // rows lr0 .. lr0 + 3
  const int64_t tile_r = tile / p.tiles_c, tile_c = tile - tile_r * p.tiles_c;
  const int64_t row0 = tile_r * 128, col0 = tile_c * 128;
  const int64_t c0 = col0 + 8 * g;
  const int nc = (int)max((int64_t)0, min((int64_t)8, p.cols - c0));
  const int nr = (int)max((int64_t)0, min((int64_t)4, p.rows - row0 - lr0));

  // a whole tile of aligned rows (the same for every thread)
  const bool whole = row0 + 128 <= p.rows && col0 + 128 <= p.cols;
  float v[4][8];
  if (p.vec_src && whole) {
    const int64_t at = (row0 + lr0) * p.ld_src + c0;
#pragma unroll
    for (int i = 0; i < 4; ++i) load8<SRC>(p.src, at + i * p.ld_src, 8, true, v[i]);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int n = i < nr ? nc : 0;
      load8<SRC>(p.src, (row0 + lr0 + i) * p.ld_src + c0, n, p.vec_src && n == 8, v[i]);
    }
  }
  if constexpr (NORM) {
    float gm[8];
    load8(p.col_mul, p.col_mul_dt, c0, nc, p.vec_mul && nc == 8, gm);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      // elements past the edges are 0 whatever the row's statistics
      const bool in = i < nr;
      normed8(v[i], in ? p.row_mul[row0 + lr0 + i] : 0.0f, gm);
      if (!whole) {
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (!in || j >= nc) v[i][j] = 0.0f;
      }
    }
  }

  if (p.colsum != nullptr) {
    // column sums in a fixed order: four rows per thread, two half warps,
    // sixteen warps
    float t[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      t[j] = (v[0][j] + v[1][j]) + (v[2][j] + v[3][j]);
      t[j] += __shfl_xor_sync(0xFFFFFFFFu, t[j], 16);
    }
    if (half == 0) {
      float4* d = reinterpret_cast<float4*>(&sm.sum[warp][8 * g]);
      d[0] = make_float4(t[0], t[1], t[2], t[3]);
      d[1] = make_float4(t[4], t[5], t[6], t[7]);
    }
  }

  // maxima of the thread's rows, columns and whole piece; infinities (rare)
  // become NaN, which maxima skip, so that the finite values set the scales
  float rm[4], cm[8], all;
  auto maxima = [&]() {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      rm[i] = max_abs(v[i][0], v[i][1], 0.0f);
#pragma unroll
      for (int j = 2; j < 8; j += 2) rm[i] = max_abs(v[i][j], v[i][j + 1], rm[i]);
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) cm[j] = max_abs(v[2][j], v[3][j], max_abs(v[0][j], v[1][j], 0.0f));
    all = max_abs(rm[2], rm[3], max_abs(rm[0], rm[1], 0.0f));
  };
  maxima();
  if (is_inf(all)) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < 8; ++j) v[i][j] = inf_to_nan(v[i][j]);
    maxima();
  }

  const int64_t rows_pad = rows_padded(p.rows), cols_pad = rows_padded(p.cols);
  uint32_t byte_all = 0;
  float inv_all = 0.0f;
  if constexpr (SQUARE) {
    const uint32_t m = warp_max_u32(__float_as_uint(all));
    if (lane == 0) sm.max[0][warp] = __uint_as_float(m);
    __syncthreads();
    byte_all = scale_byte(warp_max_u32(__float_as_uint(sm.max[0][lane & 15])));
    inv_all = inv_scale(byte_all);
  } else if (p.dst_t != nullptr) {
    uint32_t m[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      m[j] = __float_as_uint(cm[j]);
      m[j] = max(m[j], __shfl_xor_sync(0xFFFFFFFFu, m[j], 16));
    }
    if (half == 0) {
      uint4* d = reinterpret_cast<uint4*>(&sm.max[warp][8 * g]);
      d[0] = make_uint4(m[0], m[1], m[2], m[3]);
      d[1] = make_uint4(m[4], m[5], m[6], m[7]);
    }
  }

  if (p.dst != nullptr) {
    float inv[4];
    if constexpr (SQUARE) {
#pragma unroll
      for (int i = 0; i < 4; ++i) inv[i] = inv_all;
      // rows past the end, up to the next multiple of 128, have a scale too
      if (g < 4) p.sc[scale_offset(rows_pad, row0 + lr0 + g, tile_c)] = (uint8_t)byte_all;
    } else {
      // maxima of four rows over sixteen lanes: each exchange halves the rows
      // that a lane still follows, until it holds one, in four copies
      const bool b3 = lane & 8, b2 = lane & 4;
      uint32_t m[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) m[i] = __float_as_uint(rm[i]);
      const uint32_t a0 = __shfl_xor_sync(0xFFFFFFFFu, b3 ? m[0] : m[2], 8);
      const uint32_t a1 = __shfl_xor_sync(0xFFFFFFFFu, b3 ? m[1] : m[3], 8);
      const uint32_t k0 = max(b3 ? m[2] : m[0], a0), k1 = max(b3 ? m[3] : m[1], a1);
      uint32_t k = max(b2 ? k1 : k0, __shfl_xor_sync(0xFFFFFFFFu, b2 ? k0 : k1, 4));
      k = max(k, __shfl_xor_sync(0xFFFFFFFFu, k, 2));
      k = max(k, __shfl_xor_sync(0xFFFFFFFFu, k, 1));
      const uint32_t b = scale_byte(k);
      const int mine = (b3 ? 2 : 0) + (b2 ? 1 : 0);
      if ((lane & 3) == 0) p.sc[scale_offset(rows_pad, row0 + lr0 + mine, tile_c)] = (uint8_t)b;
      const float is = inv_scale(b);
#pragma unroll
      for (int i = 0; i < 4; ++i)
        inv[i] = __shfl_sync(0xFFFFFFFFu, is, (lane & 16) | ((i >> 1) << 3) | ((i & 1) << 2));
    }
    uint8_t* d = p.dst + (row0 + lr0) * p.ld_dst + c0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint2 c = codes8(v[i], inv[i]);
      if (whole) *reinterpret_cast<uint2*>(d + i * p.ld_dst) = c;
      else if (i < nr && nc > 0) store_codes8(d + i * p.ld_dst, c, nc);
    }
  }

  if (p.dst_t == nullptr && p.colsum == nullptr) return;
  __syncthreads();
  if (threadIdx.x < 128) {
    const int c = threadIdx.x;
    if (p.dst_t != nullptr) {
      uint32_t b = byte_all;
      if constexpr (!SQUARE) {
        uint32_t m = 0;
#pragma unroll
        for (int k = 0; k < 16; ++k) m = max(m, __float_as_uint(sm.max[k][c]));
        b = scale_byte(m);
        sm.inv[c] = inv_scale(b);
      }
      p.sc_t[scale_offset(cols_pad, col0 + c, tile_r)] = (uint8_t)b;
    }
    if (p.colsum != nullptr && col0 + c < p.cols) {
      float t = sm.sum[0][c];
#pragma unroll
      for (int k = 1; k < 16; ++k) t += sm.sum[k][c];
      p.colsum[tile_r * p.cols + col0 + c] = t;
    }
  }
  if (p.dst_t == nullptr) return;
  float inv[8];
  if constexpr (SQUARE) {
#pragma unroll
    for (int j = 0; j < 8; ++j) inv[j] = inv_all;
  } else {
    __syncthreads();
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const float4 x = *reinterpret_cast<const float4*>(&sm.inv[8 * g + 4 * h]);
      inv[4 * h] = x.x; inv[4 * h + 1] = x.y; inv[4 * h + 2] = x.z; inv[4 * h + 3] = x.w;
    }
  }
  // Column c is 32 words of four rows; word u lies at u ^ 2 (c / 8). A warp's
  // store (two words of sixteen columns) then covers all banks, and four
  // neighbouring words stay together, at most with their halves exchanged.
  const int u = warp * 2 + half;
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 8; j += 2) mul2(v[i][j], v[i][j + 1], inv[j], inv[j + 1], v[i][j], v[i][j + 1]);
#pragma unroll
  for (int j = 0; j < 8; ++j)
    sm.t[(8 * g + j) * 32 + (u ^ (2 * g))] = e4m3x2_sat(v[0][j], v[1][j]) | (e4m3x2_sat(v[2][j], v[3][j]) << 16);
  __syncthreads();
  const int k2 = threadIdx.x & 7;                        // sixteen rows
  const int64_t gr = row0 + 16 * k2;
#pragma unroll
  for (int it = 0; it < 2; ++it) {
    const int c = it * 64 + (threadIdx.x >> 3);
    const int64_t gc = col0 + c;
    const int cg = c >> 3;
    const uint4 x = *reinterpret_cast<const uint4*>(sm.t + c * 32 + 4 * (k2 ^ (cg >> 1)));
    const uint4 q = (cg & 1) ? make_uint4(x.z, x.w, x.x, x.y) : x;
    uint8_t* d = p.dst_t + gc * p.ld_dst_t + gr;
    if (whole) {
      *reinterpret_cast<uint4*>(d) = q;
    } else if (gc < p.cols && gr < p.rows) {
      const int64_t n = p.rows - gr;
      if (n >= 16) {
        *reinterpret_cast<uint4*>(d) = q;
      } else {
        store_codes8(d, make_uint2(q.x, q.y), (int)min(n, (int64_t)8));
        if (n > 8) store_codes8(d + 8, make_uint2(q.z, q.w), (int)n - 8);
      }
    }
  }
}

template <int SRC, bool SQUARE, bool NORM>
__global__ void __launch_bounds__(kCastThreads, 2) block_cast_kernel(CastArgs p) {
  __shared__ __align__(16) CastShared sm;
  pdl_launch_dependents();
  pdl_wait();
  cast_tile<SRC, SQUARE, NORM>(p, blockIdx.x, sm);
}

// A layer's weight and activations in one launch: the weight's tiles come
// first, so a small weight's cast hides behind the activations'.
template <int SRC_W, int SRC_X>
__global__ void __launch_bounds__(kCastThreads, 2) block_cast2_kernel(CastArgs w, CastArgs x, int w_tiles) {
  __shared__ __align__(16) CastShared sm;
  pdl_launch_dependents();
  pdl_wait();
  if ((int)blockIdx.x < w_tiles) cast_tile<SRC_W, true, false>(w, blockIdx.x, sm);
  else cast_tile<SRC_X, false, false>(x, (int64_t)blockIdx.x - w_tiles, sm);
}

struct DequantArgs {
  const uint8_t* src; int64_t ld; const uint8_t* sc;
  int64_t rows, cols; void* dst; int64_t ld_dst;
  int vec_dst;
  uint32_t chunks;   // 8-element chunks per row
};

// Eight codes per thread and step, so a warp's stores cover whole lines; four
// steps under way together. I: the type that counts chunks (64-bit division
// costs as much as the conversion).
template <int DST, class I>
__global__ void __launch_bounds__(256) block_dequant_kernel(DequantArgs p) {
  pdl_launch_dependents();
  pdl_wait();
  const I total = (I)p.rows * p.chunks;
  const int64_t rows_pad = rows_padded(p.rows);
  const I first = (I)blockIdx.x * 1024 + threadIdx.x;
  uint2 q[4];
  uint32_t b[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const I e = first + 256 * k;
    if (e < total) {
      const I r = e / p.chunks;
      const int c0 = (int)(e - r * p.chunks) * 8;
      q[k] = *reinterpret_cast<const uint2*>(p.src + (int64_t)r * p.ld + c0);     // rows are padded to 16 codes
      b[k] = p.sc[scale_offset(rows_pad, (int64_t)r, c0 >> 7)];
    }
  }
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const I e = first + 256 * k;
    if (e < total) {
      const I r = e / p.chunks;
      const int c0 = (int)(e - r * p.chunks) * 8;
      const float s = scale_value(b[k]);
      const uint32_t w[2] = {q[k].x, q[k].y};
      float v[8];
#pragma unroll
      for (int h = 0; h < 4; ++h) {
        const uint32_t f = f16x2_from_e4m3x2((w[h >> 1] >> (16 * (h & 1))) & 0xFFFFu);
        mul2(f16lo_to_f32(f), f16hi_to_f32(f), s, s, v[2 * h], v[2 * h + 1]);
      }
      const int n = (int)min((int64_t)8, p.cols - c0);
      store8<DST>(p.dst, (int64_t)r * p.ld_dst + c0, n, p.vec_dst && n == 8, v);
    }
  }
}

CastArgs cast_args(const void* src, int es, int64_t rows, int64_t cols, int64_t ld_src, const float* row_mul,
                   const void* col_mul, int col_mul_dt, void* dst, int64_t ld_dst, void* sc, void* dst_t,
                   int64_t ld_dst_t, void* sc_t, float* colsum) {
  return CastArgs{src, rows, cols, ld_src, row_mul, col_mul, col_mul_dt, static_cast<uint8_t*>(dst), ld_dst,
                  static_cast<uint8_t*>(sc), static_cast<uint8_t*>(dst_t), ld_dst_t, static_cast<uint8_t*>(sc_t),
                  colsum,
                  vec16(src, ld_src, es) ? 1 : 0, vec16(col_mul, 8, 4) ? 1 : 0, (cols + 127) / 128};
}

int64_t cast_tiles(int64_t rows, int64_t cols) { return ((rows + 127) / 128) * ((cols + 127) / 128); }

// The weight (square scales) and the activations of a layer, both checked.
int cast_pair(const CastArgs& w, int w_dt, const CastArgs& x, int x_dt, cudaStream_t s) {
  const int64_t tw = cast_tiles(w.rows, w.cols), tx = cast_tiles(x.rows, x.cols);
  if (tw + tx > (1ll << 31) - 1) return APA_ERR_INVALID;
  void (*k)(CastArgs, CastArgs, int) = nullptr;
#define APA_CAST2_CASE(W)                                                       \
  k = x_dt == APA_DT_F32   ? block_cast2_kernel<W, APA_DT_F32>                  \
      : x_dt == APA_DT_F16 ? block_cast2_kernel<W, APA_DT_F16>                  \
                           : block_cast2_kernel<W, APA_DT_BF16>
  if (w_dt == APA_DT_F32) APA_CAST2_CASE(APA_DT_F32);
  else if (w_dt == APA_DT_F16) APA_CAST2_CASE(APA_DT_F16);
  else APA_CAST2_CASE(APA_DT_BF16);
#undef APA_CAST2_CASE
  return launch_kernel(k, dim3((unsigned)(tw + tx)), dim3(kCastThreads), 0, s, 1, w, x, (int)tw) == cudaSuccess
             ? APA_OK : APA_ERR_CUDA;
}

// Column sums of [parts, cols] fp32 partials in a fixed order, rounded once to
// the output's type. A CTA has 8 columns (one sector of every row) and 16, 64 or
// 128 threads for each, so a few hundred to a thousand rows are one or two
// rounds of loads.
__global__ void __launch_bounds__(1024) block_colsum_kernel(const float* part, int64_t parts, int64_t cols, void* out,
                                                            int out_dt) {
  pdl_launch_dependents();
  pdl_wait();
  __shared__ float s[32][8];
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  const int64_t c = (int64_t)blockIdx.x * 8 + (lane & 7);
  const int per = blockDim.x >> 3;
  float t = 0.0f;
  if (c < cols) {
    int64_t r = threadIdx.x >> 3;
    for (; r + 7 * per < parts; r += 8 * per) {
      float x[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) x[k] = part[(r + per * k) * cols + c];
#pragma unroll
      for (int k = 0; k < 8; ++k) t += x[k];
    }
    float x[7];
#pragma unroll
    for (int k = 0; k < 7; ++k) x[k] = r + per * k < parts ? part[(r + per * k) * cols + c] : 0.0f;
#pragma unroll
    for (int k = 0; k < 7; ++k) t += x[k];
  }
  t += __shfl_xor_sync(0xFFFFFFFFu, t, 8);
  t += __shfl_xor_sync(0xFFFFFFFFu, t, 16);
  if (lane < 8) s[w][lane] = t;
  __syncthreads();
  if (w == 0) {
    const int warps = blockDim.x >> 5;
    float u = 0.0f;
    for (int k = lane >> 3; k < warps; k += 4) u += s[k][lane & 7];
    u += __shfl_xor_sync(0xFFFFFFFFu, u, 8);
    u += __shfl_xor_sync(0xFFFFFFFFu, u, 16);
    if (lane < 8 && c < cols) from_f32(out, out_dt, c, u);
  }
}

int launch_colsum(const float* part, int64_t parts, int64_t cols, void* out, int out_dt, cudaStream_t s) {
  const int64_t grid = (cols + 7) / 8;
  const int threads = parts <= 32 ? 128 : parts <= 256 ? 512 : 1024;
  return launch_kernel(block_colsum_kernel, dim3((unsigned)grid), dim3(threads), 0, s, 1, part, parts, cols, out,
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
  const CastArgs a = cast_args(src, es, rows, cols, ld_src, row_mul, col_mul, col_mul_dtype, dst, ld_dst, scales, dst_t,
                               ld_dst_t, scales_t, colsum_partial);
  void (*k)(CastArgs);
  const bool norm = row_mul != nullptr;
#define APA_CAST_CASE(SRC)                                                                        \
  k = square ? (norm ? block_cast_kernel<SRC, true, true> : block_cast_kernel<SRC, true, false>)  \
             : (norm ? block_cast_kernel<SRC, false, true> : block_cast_kernel<SRC, false, false>)
  if (src_dtype == APA_DT_F32) APA_CAST_CASE(APA_DT_F32);
  else if (src_dtype == APA_DT_F16) APA_CAST_CASE(APA_DT_F16);
  else APA_CAST_CASE(APA_DT_BF16);
#undef APA_CAST_CASE
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
                vec16(dst, ld_dst, es) ? 1 : 0, (uint32_t)((cols + 7) / 8)};
  const int64_t total = rows * (int64_t)a.chunks, grid = (total + 1023) / 1024;
  if (grid > (1ll << 31) - 1) return APA_ERR_INVALID;
  const bool wide = total > (1ll << 31) - 2048;
  void (*k)(DequantArgs);
#define APA_DEQUANT_CASE(DST) k = wide ? block_dequant_kernel<DST, uint64_t> : block_dequant_kernel<DST, uint32_t>
  if (dst_dtype == APA_DT_F32) APA_DEQUANT_CASE(APA_DT_F32);
  else if (dst_dtype == APA_DT_F16) APA_DEQUANT_CASE(APA_DT_F16);
  else APA_DEQUANT_CASE(APA_DT_BF16);
#undef APA_DEQUANT_CASE
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
