// Root-mean-square norm with the residual's addition, forward and backward.
//
//   r    = RN(x + residual)                    the residual stream, x's type
//   rstd = (mean_k r^2 + eps)^(-1/2)           fp32
//   y    = r rstd gamma                        x's type, or an E4M3 block
//                                              tensor (rows form)
//   dx   = rstd (gamma dy - xhat mean_k(gamma dy xhat)) + dr,  xhat = r rstd
//   dgamma = sum_rows dy xhat
//
// The statistics are those of the stored stream r (not of the unrounded sum),
// so the backward, which reads r back, differentiates the function the
// forward computed. dx is the gradient of x and of the residual alike.
//
// Bound by HBM: a row is read once into registers (TPR threads per row, NV
// chunks of eight elements per thread), reduced, and written once. A block of
// 128 columns is sixteen neighbouring lanes, so its maximum is four shuffles.
// The backward keeps the columns' dgamma sums in registers over all rows of a
// CTA and writes them once, so a second kernel adds only a few hundred
// partial rows, in a fixed order.
#include "block_scale.cuh"

namespace apa {
namespace blk {

int launch_colsum(const float* part, int64_t parts, int64_t cols, void* out, int out_dt, cudaStream_t s);

struct NormArgs {
  const void* x; int64_t ld_x;
  const void* res; int64_t ld_res;
  const void* gamma; int gamma_dt;
  void* r; int64_t ld_r;          // stored stream (null: x is the stream)
  void* y; int64_t ld_y;          // plain output, or
  uint8_t* q; int64_t ld_q; uint8_t* sc;
  float* rstd;
  int64_t rows, cols;
  float eps;
  int vec_x, vec_res, vec_r, vec_y;
};

template <int TPR>
constexpr int norm_threads() { return TPR < 128 ? 128 : TPR; }

// Sum over the TPR threads of a row; every thread gets it.
template <int TPR>
__device__ __forceinline__ float row_sum(float v, float* s_red) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, o);
  if constexpr (TPR > 32) {
    // one row per CTA
    constexpr int kWarps = TPR / 32;
    __syncthreads();   // s_red is free again
    if ((threadIdx.x & 31) == 0) s_red[threadIdx.x >> 5] = v;
    __syncthreads();
    float t = (threadIdx.x & 31) < kWarps ? s_red[threadIdx.x & 31] : 0.0f;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) t += __shfl_xor_sync(0xFFFFFFFFu, t, o);
    v = t;
  }
  return v;
}

// a^(-1/2) to within an ulp: one Newton step on the hardware's approximation
// (which alone is good to two ulps).
__device__ __forceinline__ float rsqrt_refined(float a) {
  const float y = rsqrtf(a);
  if (!(a > 0.0f) || a > 3.0e38f) return y;
  const float h = a * y;
  const float e = __fmaf_rn(-h, y, __fmaf_rn(__fmaf_rn(a, y, -h), -y, 1.0f));
  return __fmaf_rn(0.5f * y, e, y);
}

template <int DT, int TPR, int NV, bool QUANT>
__global__ void __launch_bounds__(norm_threads<TPR>()) rmsnorm_kernel(NormArgs p) {
  constexpr int kRows = norm_threads<TPR>() / TPR;
  __shared__ float s_red[32];
  pdl_launch_dependents();
  pdl_wait();
  const int t = threadIdx.x % TPR;
  const int64_t row = (int64_t)blockIdx.x * kRows + threadIdx.x / TPR;
  if (TPR == 32 && row >= p.rows) return;      // a whole warp
  float v[NV][8];
  float ss = 0.0f;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int64_t c0 = ((int64_t)t + (int64_t)TPR * i) * 8;
    const int n = (int)max((int64_t)0, min((int64_t)8, p.cols - c0));
    load8<DT>(p.x, row * p.ld_x + c0, n, p.vec_x && n == 8, v[i]);
    if (p.res != nullptr) {
      float u[8];
      load8<DT>(p.res, row * p.ld_res + c0, n, p.vec_res && n == 8, u);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        v[i][j] += u[j];
        if constexpr (DT == APA_DT_F16) v[i][j] = f16_to_f32(f16_from_f32(v[i][j]));
        if constexpr (DT == APA_DT_BF16) v[i][j] = bf16_to_f32(bf16_from_f32(v[i][j]));
      }
      if (n > 0) store8<DT>(p.r, row * p.ld_r + c0, n, p.vec_r && n == 8, v[i]);
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) ss = __fmaf_rn(v[i][j], v[i][j], ss);
  }
  ss = row_sum<TPR>(ss, s_red);
  const float rstd = rsqrt_refined(ss / (float)p.cols + p.eps);
  if (t == 0 && p.rstd != nullptr) p.rstd[row] = rstd;
  const int64_t rows_pad = rows_padded(p.rows);
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int64_t c0 = ((int64_t)t + (int64_t)TPR * i) * 8;
    const int n = (int)max((int64_t)0, min((int64_t)8, p.cols - c0));
    float y[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) y[j] = j < n ? normed(v[i][j], rstd, to_f32(p.gamma, p.gamma_dt, c0 + j)) : 0.0f;
    if constexpr (QUANT) {
      uint32_t m = 0;
#pragma unroll
      for (int j = 0; j < 8; ++j) m = max(m, mag_bits(y[j]));
      const bool odd = bits_nonfinite(m);
      if (odd) {
        m = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) m = max(m, finite_mag(y[j]));
      }
#pragma unroll
      for (int o = 8; o > 0; o >>= 1) m = max(m, __shfl_xor_sync(0xFFFFFFFFu, m, o));
      const uint32_t b = scale_byte(m);
      const float is = inv_scale(b);
      if (n > 0) {
        uint2 w;
        w.x = codes2(y[0] * is, y[1] * is, odd) | (codes2(y[2] * is, y[3] * is, odd) << 16);
        w.y = codes2(y[4] * is, y[5] * is, odd) | (codes2(y[6] * is, y[7] * is, odd) << 16);
        store_codes8(p.q + row * p.ld_q + c0, w, n);
        if ((t & 15) == 0) p.sc[scale_offset(rows_pad, row, c0 >> 7)] = (uint8_t)b;
      }
    } else {
      if (n > 0) store8<DT>(p.y, row * p.ld_y + c0, n, p.vec_y && n == 8, y);
    }
  }
}

struct NormBwdArgs {
  const void* dy; int64_t ld_dy;
  const void* r; int64_t ld_r;
  const float* rstd;
  const void* gamma; int gamma_dt;
  const void* dr; int64_t ld_dr;     // nullable: gradient of the stream
  void* dx; int64_t ld_dx;
  float* part;                       // [grid, cols] dgamma partials
  int64_t rows, cols;
  int vec_dy, vec_r, vec_dr, vec_dx;
};

template <int DT, int TPR, int NV>
__global__ void __launch_bounds__(norm_threads<TPR>()) rmsnorm_bwd_kernel(NormBwdArgs p) {
  constexpr int kRows = norm_threads<TPR>() / TPR;
  __shared__ float s_red[32];
  extern __shared__ float s_dg[];    // kRows > 1: [kRows][NV * TPR * 8]
  pdl_launch_dependents();
  pdl_wait();
  const int t = threadIdx.x % TPR, sub = threadIdx.x / TPR;
  float dg[NV][8], gm[NV][8];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int64_t c0 = ((int64_t)t + (int64_t)TPR * i) * 8;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      dg[i][j] = 0.0f;
      gm[i][j] = c0 + j < p.cols ? to_f32(p.gamma, p.gamma_dt, c0 + j) : 0.0f;
    }
  }
  const float inv_n = 1.0f / (float)p.cols;
  for (int64_t row = (int64_t)blockIdx.x * kRows + sub; row < p.rows; row += (int64_t)gridDim.x * kRows) {
    const float rstd = p.rstd[row];
    float dy[NV][8], xh[NV][8];
    float s = 0.0f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int64_t c0 = ((int64_t)t + (int64_t)TPR * i) * 8;
      const int n = (int)max((int64_t)0, min((int64_t)8, p.cols - c0));
      load8<DT>(p.dy, row * p.ld_dy + c0, n, p.vec_dy && n == 8, dy[i]);
      load8<DT>(p.r, row * p.ld_r + c0, n, p.vec_r && n == 8, xh[i]);
    }
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        xh[i][j] *= rstd;
        dg[i][j] = __fmaf_rn(dy[i][j], xh[i][j], dg[i][j]);
        dy[i][j] *= gm[i][j];
        s = __fmaf_rn(dy[i][j], xh[i][j], s);
      }
    const float c = row_sum<TPR>(s, s_red) * inv_n;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int64_t c0 = ((int64_t)t + (int64_t)TPR * i) * 8;
      const int n = (int)max((int64_t)0, min((int64_t)8, p.cols - c0));
      float o[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) o[j] = rstd * __fmaf_rn(-xh[i][j], c, dy[i][j]);
      if (p.dr != nullptr) {
        float u[8];
        load8<DT>(p.dr, row * p.ld_dr + c0, n, p.vec_dr && n == 8, u);
#pragma unroll
        for (int j = 0; j < 8; ++j) o[j] += u[j];
      }
      if (n > 0) store8<DT>(p.dx, row * p.ld_dx + c0, n, p.vec_dx && n == 8, o);
    }
  }
  float* out = p.part + (int64_t)blockIdx.x * p.cols;
  if constexpr (kRows > 1) {
    constexpr int kW = NV * TPR * 8;
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int j = 0; j < 8; ++j) s_dg[sub * kW + (t + TPR * i) * 8 + j] = dg[i][j];
    __syncthreads();
    for (int c = threadIdx.x; c < kW && c < p.cols; c += norm_threads<TPR>()) {
      float a = s_dg[c];
#pragma unroll
      for (int k = 1; k < kRows; ++k) a += s_dg[k * kW + c];
      out[c] = a;
    }
  } else {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int64_t c0 = ((int64_t)t + (int64_t)TPR * i) * 8;
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (c0 + j < p.cols) out[c0 + j] = dg[i][j];
    }
  }
}

constexpr int64_t kMaxNormCols = 32768;   // 1024 threads x 4 chunks of eight

// Threads per row and chunks per thread: a warp per row up to 1024 columns
// (no block-wide sum), then 128, 512 and 1024 threads with at most four
// chunks, which keeps a row in 32 registers per thread.
template <template <int, int, int> class L, int DT, class A>
int norm_dispatch(const A& a, cudaStream_t s) {
  const int64_t chunks = (a.cols + 7) / 8;
  if (chunks <= 32) return L<DT, 32, 1>::run(a, s);
  if (chunks <= 64) return L<DT, 32, 2>::run(a, s);
  if (chunks <= 128) return L<DT, 32, 4>::run(a, s);
  if (chunks <= 256) return L<DT, 128, 2>::run(a, s);
  if (chunks <= 512) return L<DT, 128, 4>::run(a, s);
  if (chunks <= 1024) return L<DT, 512, 2>::run(a, s);
  if (chunks <= 2048) return L<DT, 512, 4>::run(a, s);
  return L<DT, 1024, 4>::run(a, s);
}

template <int DT, int TPR, int NV> struct NormFwd {
  static int run(const NormArgs& a, cudaStream_t s) {
    constexpr int kRows = norm_threads<TPR>() / TPR;
    const int64_t grid = (a.rows + kRows - 1) / kRows;
    void (*k)(NormArgs) = a.q ? rmsnorm_kernel<DT, TPR, NV, true> : rmsnorm_kernel<DT, TPR, NV, false>;
    return launch_kernel(k, dim3((unsigned)grid), dim3(norm_threads<TPR>()), 0, s, 1, a) == cudaSuccess ? APA_OK
                                                                                                        : APA_ERR_CUDA;
  }
};

template <int TPR>
int64_t norm_bwd_grid(int64_t rows) {
  constexpr int kRows = norm_threads<TPR>() / TPR;
  const int64_t per_sm = TPR >= 1024 ? 1 : TPR >= 512 ? 2 : 6;
  return std::min<int64_t>((rows + kRows - 1) / kRows, per_sm * num_sms());
}

template <int DT, int TPR, int NV> struct NormBwd {
  static int run(const NormBwdArgs& a, cudaStream_t s) {
    constexpr int kRows = norm_threads<TPR>() / TPR;
    const size_t smem = kRows > 1 ? (size_t)kRows * NV * TPR * 8 * 4 : 0;   // at most 16 KB
    return launch_kernel(rmsnorm_bwd_kernel<DT, TPR, NV>, dim3((unsigned)norm_bwd_grid<TPR>(a.rows)),
                         dim3(norm_threads<TPR>()), smem, s, 1, a) == cudaSuccess ? APA_OK : APA_ERR_CUDA;
  }
};

// CTAs (= dgamma partial rows) of the backward
int64_t norm_bwd_parts(int64_t rows, int64_t cols) {
  const int64_t chunks = (cols + 7) / 8;
  if (chunks <= 128) return norm_bwd_grid<32>(rows);
  if (chunks <= 512) return norm_bwd_grid<128>(rows);
  if (chunks <= 2048) return norm_bwd_grid<512>(rows);
  return norm_bwd_grid<1024>(rows);
}

int norm_dims(int64_t rows, int64_t cols) {
  if (rows <= 0 || cols <= 0 || rows > (1ll << 31) - 256) return APA_ERR_INVALID;
  return cols > kMaxNormCols ? APA_ERR_UNSUPPORTED : APA_OK;
}

}  // namespace blk
}  // namespace apa

extern "C" int apa_rmsnorm_fwd(const void* x, int64_t ld_x, const void* residual, int64_t ld_res, const void* gamma,
                               int gamma_dtype, int dtype, int64_t rows, int64_t cols, float eps, void* stream_out,
                               int64_t ld_stream, void* y, int64_t ld_y, void* q, int64_t ld_q, void* scales,
                               float* rstd, void* stream) {
  using namespace apa::blk;
  if (!x || !gamma) return APA_ERR_INVALID;
  if (int st = norm_dims(rows, cols)) return st;
  const int es = elem_bytes(dtype);
  if (es == 0 || elem_bytes(gamma_dtype) == 0) return APA_ERR_UNSUPPORTED;
  if (ld_x < cols || (residual && ld_res < cols)) return APA_ERR_INVALID;
  if ((residual == nullptr) != (stream_out == nullptr) || (stream_out && ld_stream < cols)) return APA_ERR_INVALID;
  if ((y == nullptr) == (q == nullptr) || (y && ld_y < cols)) return APA_ERR_INVALID;   // one output or the other
  if ((q == nullptr) != (scales == nullptr) || (q && ld_q < cols)) return APA_ERR_INVALID;
  if (q && !vec16(q, ld_q, 1)) return APA_ERR_ALIGN;
  NormArgs a{x, ld_x, residual, ld_res, gamma, gamma_dtype, stream_out, ld_stream, y, ld_y,
             static_cast<uint8_t*>(q), ld_q, static_cast<uint8_t*>(scales), rstd, rows, cols, eps,
             vec16(x, ld_x, es) ? 1 : 0, residual && vec16(residual, ld_res, es) ? 1 : 0,
             stream_out && vec16(stream_out, ld_stream, es) ? 1 : 0, y && vec16(y, ld_y, es) ? 1 : 0};
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (dtype == APA_DT_F32) return norm_dispatch<NormFwd, APA_DT_F32>(a, s);
  if (dtype == APA_DT_F16) return norm_dispatch<NormFwd, APA_DT_F16>(a, s);
  return norm_dispatch<NormFwd, APA_DT_BF16>(a, s);
}

extern "C" int apa_rmsnorm_bwd_workspace(int64_t rows, int64_t cols, int64_t* bytes_out) {
  using namespace apa::blk;
  if (!bytes_out) return APA_ERR_INVALID;
  if (int st = norm_dims(rows, cols)) return st;
  *bytes_out = norm_bwd_parts(rows, cols) * cols * 4;
  return APA_OK;
}

extern "C" int apa_rmsnorm_bwd(const void* dy, int64_t ld_dy, const void* r, int64_t ld_r, const float* rstd,
                               const void* gamma, int gamma_dtype, const void* dr, int64_t ld_dr, void* dx,
                               int64_t ld_dx, int dtype, int64_t rows, int64_t cols, void* dgamma, void* workspace,
                               int64_t workspace_bytes, void* stream) {
  using namespace apa::blk;
  if (!dy || !r || !rstd || !gamma || !dx || !dgamma || !workspace) return APA_ERR_INVALID;
  if (int st = norm_dims(rows, cols)) return st;
  const int es = elem_bytes(dtype);
  if (es == 0 || elem_bytes(gamma_dtype) == 0) return APA_ERR_UNSUPPORTED;
  if (ld_dy < cols || ld_r < cols || ld_dx < cols || (dr && ld_dr < cols)) return APA_ERR_INVALID;
  if ((reinterpret_cast<uintptr_t>(workspace) & 15u) != 0) return APA_ERR_ALIGN;
  const int64_t parts = norm_bwd_parts(rows, cols);
  if (workspace_bytes < parts * cols * 4) return APA_ERR_INVALID;
  NormBwdArgs a{dy, ld_dy, r, ld_r, rstd, gamma, gamma_dtype, dr, ld_dr, dx, ld_dx, static_cast<float*>(workspace),
                rows, cols, vec16(dy, ld_dy, es) ? 1 : 0, vec16(r, ld_r, es) ? 1 : 0,
                dr && vec16(dr, ld_dr, es) ? 1 : 0, vec16(dx, ld_dx, es) ? 1 : 0};
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  int st;
  if (dtype == APA_DT_F32) st = norm_dispatch<NormBwd, APA_DT_F32>(a, s);
  else if (dtype == APA_DT_F16) st = norm_dispatch<NormBwd, APA_DT_F16>(a, s);
  else st = norm_dispatch<NormBwd, APA_DT_BF16>(a, s);
  if (st != APA_OK) return st;
  return launch_colsum(a.part, parts, cols, dgamma, gamma_dtype, s);
}
