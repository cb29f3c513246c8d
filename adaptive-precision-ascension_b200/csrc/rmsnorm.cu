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
// Bound by HBM. CTAs are persistent: TPR threads share a row, NV chunks of
// eight elements each, and every thread copies its own chunks of the rows to
// come into shared memory with cp.async, two rows ahead (no barrier: it reads
// only what it copied). So loads are in flight while a row is reduced and
// stored; without that the row's two block-wide barriers left HBM at half its
// rate. A block of 128 columns is sixteen neighbouring lanes, so its maximum is
// four shuffles. The backward keeps the columns' dgamma sums in registers over
// all rows of a CTA and writes them once; a second kernel adds these few hundred
// partial rows in a fixed order.
//
// Measured on a B200, inputs in HBM (us, TB/s of what is read and written):
// 8192 x 4096 bf16 forward 21.0, 6.4; with residual 48, 5.6; residual to E4M3
// 43, 5.4; backward 53, 3.8, with the stream's gradient 61, 4.4; 33280 x 512
// fp32 forward 21.9, 6.2, backward 39.7, 5.2. The backward is short of HBM's
// rate by the latency of a row's steps (issue slots 51 % busy, the waits spread
// over shared memory, gamma and the barriers). Neither a row's rstd loaded a row
// ahead nor gamma in registers changed that by more than 4 %: more threads per
// SM would, but registers hold the columns' sums.
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
  int vec_x, vec_res, vec_r, vec_y, vec_g;
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

template <int DT> constexpr int pieces() { return DT == APA_DT_F32 ? 2 : 1; }   // 16-byte pieces per chunk

// The chunks of one thread in one row, in planes of 16 bytes per thread (so a
// warp's accesses are conflict-free). at: this thread's bytes of plane 0.
template <int DT, int TPR, int NV>
__device__ __forceinline__ void fetch_row(uint32_t at, const void* p, int64_t row_at, int t, int cols) {
  constexpr int ES = DT == APA_DT_F32 ? 4 : 2;
  const char* row = static_cast<const char*>(p) + row_at * ES;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c0 = (t + TPR * i) * 8;
    if (c0 < cols) {
      const char* g = row + c0 * ES;
#pragma unroll
      for (int k = 0; k < pieces<DT>(); ++k)
        cp_async16(at + (uint32_t)((i * pieces<DT>() + k) * norm_threads<TPR>() * 16), g + 16 * k);
    }
  }
}

// Chunk i of the row: from shared memory (ASYNC, whole chunks only) or memory.
template <int DT, int TPR, bool ASYNC>
__device__ __forceinline__ void chunk8(const char* at, int i, const void* p, int64_t from, int n, bool vec,
                                       float (&v)[8]) {
  if constexpr (ASYNC) {
    if (n > 0) {
      const char* a = at + i * pieces<DT>() * norm_threads<TPR>() * 16;
      const uint4 x = *reinterpret_cast<const uint4*>(a);
      if constexpr (DT == APA_DT_F32) {
        const uint4 y = *reinterpret_cast<const uint4*>(a + norm_threads<TPR>() * 16);
        v[0] = __uint_as_float(x.x); v[1] = __uint_as_float(x.y);
        v[2] = __uint_as_float(x.z); v[3] = __uint_as_float(x.w);
        v[4] = __uint_as_float(y.x); v[5] = __uint_as_float(y.y);
        v[6] = __uint_as_float(y.z); v[7] = __uint_as_float(y.w);
      } else {
        unpack8<DT>(x, v);
      }
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = 0.0f;
    }
  } else {
    load8<DT>(p, from, n, vec && n == 8, v);
  }
}

// Rows in flight: three (or two) row buffers where they fit two CTAs (or one)
// on an SM, else none.
constexpr int norm_depth(int slot_bytes) {
  return 3 * slot_bytes <= 75 * 1024 ? 3 : 2 * slot_bytes <= 200 * 1024 ? 2 : 0;
}

template <int DT, int TPR, int NV> struct NormCfg {
  static constexpr int kThreads = norm_threads<TPR>();
  static constexpr int kRows = kThreads / TPR;
  static constexpr int kPlane = kThreads * 16;
  static constexpr int kArray = NV * pieces<DT>() * kPlane;
  static constexpr int kSlot = 2 * kArray;                       // x, residual
  static constexpr int kDepth = norm_depth(kSlot);
};

template <int DT, int TPR, int NV, bool QUANT, bool ASYNC>
__global__ void __launch_bounds__(norm_threads<TPR>()) rmsnorm_kernel(NormArgs p) {
  using C = NormCfg<DT, TPR, NV>;
  constexpr int kRows = C::kRows;
  constexpr int D = ASYNC ? C::kDepth : 1;
  constexpr int ES = DT == APA_DT_F32 ? 4 : 2;
  __shared__ float s_red[32];
  extern __shared__ __align__(16) char s_rows[];
  pdl_launch_dependents();
  pdl_wait();
  const int t = threadIdx.x % TPR;
  const int cols = (int)p.cols;
  const int64_t step = (int64_t)gridDim.x * kRows;
  const int64_t rows_pad = rows_padded(p.rows);
  char* mine = s_rows + threadIdx.x * 16;
  auto fetch = [&](int64_t row, int slot) {
    if constexpr (ASYNC) {
      if (row < p.rows) {
        const uint32_t at = static_cast<uint32_t>(__cvta_generic_to_shared(mine + slot * C::kSlot));
        fetch_row<DT, TPR, NV>(at, p.x, row * p.ld_x, t, cols);
        if (p.res != nullptr) fetch_row<DT, TPR, NV>(at + C::kArray, p.res, row * p.ld_res, t, cols);
      }
      cp_async_commit();
    }
  };
  // this thread's elements in chunk i (whole chunks or none with ASYNC)
  auto count = [&](int i) {
    const int left = cols - (t + TPR * i) * 8;
    return ASYNC ? (left > 0 ? 8 : 0) : max(0, min(8, left));
  };
  // a persistent CTA keeps the weight in registers
  float gm[NV][8];
  if constexpr (ASYNC) {
#pragma unroll
    for (int i = 0; i < NV; ++i)
      load8(p.gamma, p.gamma_dt, (t + TPR * i) * 8, count(i), p.vec_g && count(i) == 8, gm[i]);
  }
  int64_t row = (int64_t)blockIdx.x * kRows + threadIdx.x / TPR;
#pragma unroll
  for (int d = 0; d < D - 1; ++d) fetch(row + d * step, d);
  int slot = 0;
  // TPR > 32: a CTA's threads share every row, so the loop is uniform
  for (; row < p.rows; row += step) {
    if constexpr (ASYNC) {
      fetch(row + (D - 1) * step, slot == 0 ? D - 1 : slot - 1);
      cp_async_wait<D - 1>();
    }
    const char* at = mine + slot * C::kSlot;
    const char* x_row = static_cast<const char*>(p.x) + row * p.ld_x * ES;
    const char* res_row = static_cast<const char*>(p.res) + row * p.ld_res * ES;
    char* r_row = static_cast<char*>(p.r) + row * p.ld_r * ES;
    float v[NV][8];
    float ss = 0.0f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c0 = (t + TPR * i) * 8;
      const int n = count(i);
      chunk8<DT, TPR, ASYNC>(at, i, x_row, c0, n, p.vec_x, v[i]);
      if (p.res != nullptr) {
        float u[8];
        chunk8<DT, TPR, ASYNC>(at + C::kArray, i, res_row, c0, n, p.vec_res, u);
#pragma unroll
        for (int j = 0; j < 8; ++j) v[i][j] += u[j];
        if constexpr (DT == APA_DT_F32) {
          if (n > 0) store8<DT>(r_row, c0, n, p.vec_r && n == 8, v[i]);
        } else {
          const uint4 w = pack8<DT>(v[i]);
          unpack8<DT>(w, v[i]);
          if (p.vec_r && n == 8) *reinterpret_cast<uint4*>(r_row + c0 * ES) = w;
          else if (n > 0) store8<DT>(r_row, c0, n, false, v[i]);
        }
      }
      // squares in two chains per chunk, then the chunks, then the threads
      float q0 = 0.0f, q1 = 0.0f;
#pragma unroll
      for (int j = 0; j < 8; j += 2) fma2(v[i][j], v[i][j + 1], v[i][j], v[i][j + 1], q0, q1, q0, q1);
      ss += q0 + q1;
    }
    ss = row_sum<TPR>(ss, s_red);
    const float rstd = rsqrt_refined(ss / (float)cols + p.eps);
    if (t == 0 && p.rstd != nullptr) p.rstd[row] = rstd;
    uint8_t* q_row = p.q + row * p.ld_q;
    char* y_row = static_cast<char*>(p.y) + row * p.ld_y * ES;
    uint8_t* sc_row = p.sc + scale_offset(rows_pad, row, 0);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c0 = (t + TPR * i) * 8;
      const int n = count(i);
      float (&y)[8] = v[i];
      if constexpr (ASYNC) {
        normed8(y, rstd, gm[i]);
      } else {
        load8(p.gamma, p.gamma_dt, c0, n, p.vec_g && n == 8, gm[i]);
        normed8(y, rstd, gm[i]);
      }
      if (n < 8) {
        // columns past the end are 0 whatever the row's statistics
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (j >= n) y[j] = 0.0f;
      }
      if constexpr (QUANT) {
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
        if (n > 0) {
          const uint2 w = codes8(y, inv_scale(b));
          if (ASYNC || n == 8) *reinterpret_cast<uint2*>(q_row + c0) = w;
          else store_codes8(q_row + c0, w, n);
          // byte kb % 4 of the word of group kb / 4
          if ((t & 15) == 0) sc_row[(int64_t)(c0 >> 9) * rows_pad * 4 + ((c0 >> 7) & 3)] = (uint8_t)b;
        }
      } else {
        if (n > 0) store8<DT>(y_row, c0, n, p.vec_y && n == 8, y);
      }
    }
    if constexpr (ASYNC) slot = slot + 1 == D ? 0 : slot + 1;
  }
  if constexpr (ASYNC) cp_async_wait<0>();
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
  int vec_dy, vec_r, vec_dr, vec_dx, vec_g;
};

// CTAs of the backward per SM, which is what bounds a thread's registers.
constexpr int norm_bwd_resident(int tpr, int nv) {
  return tpr >= 512 ? 1 : tpr == 256 ? 3 : tpr == 128 && nv == 1 ? 8 : 4;
}

template <int DT, int DY, int TPR, int NV> struct NormBwdCfg {
  static constexpr int kThreads = norm_threads<TPR>();
  static constexpr int kRows = kThreads / TPR;
  static constexpr int kPlane = kThreads * 16;
  static constexpr int kArray = NV * pieces<DT>() * kPlane;
  static constexpr int kArrayDy = NV * pieces<DY>() * kPlane;
  static constexpr int kSlot = kArrayDy + 2 * kArray;            // dy; r, dr
  static constexpr int kDepth = norm_depth(kSlot);
  static constexpr int kSums = kRows > 1 ? kRows * NV * TPR * 8 * 4 : 0;
};

template <int DT, int DY, int TPR, int NV, bool ASYNC>
__global__ void __launch_bounds__(norm_threads<TPR>(), norm_bwd_resident(TPR, NV)) rmsnorm_bwd_kernel(NormBwdArgs p) {
  using C = NormBwdCfg<DT, DY, TPR, NV>;
  constexpr int kRows = C::kRows;
  constexpr int D = ASYNC ? C::kDepth : 1;
  constexpr int ES = DT == APA_DT_F32 ? 4 : 2, EY = DY == APA_DT_F32 ? 4 : 2;
  const int cols = (int)p.cols;
  __shared__ float s_red[32];
  extern __shared__ __align__(16) char s_rows[];    // row buffers, then [kRows][NV * TPR * 8] sums
  pdl_launch_dependents();
  pdl_wait();
  const int t = threadIdx.x % TPR, sub = threadIdx.x / TPR;
  const int64_t step = (int64_t)gridDim.x * kRows;
  char* mine = s_rows + threadIdx.x * 16;
  auto fetch = [&](int64_t row, int slot) {
    if constexpr (ASYNC) {
      if (row < p.rows) {
        const uint32_t at = static_cast<uint32_t>(__cvta_generic_to_shared(mine + slot * C::kSlot));
        fetch_row<DY, TPR, NV>(at, p.dy, row * p.ld_dy, t, cols);
        fetch_row<DT, TPR, NV>(at + C::kArrayDy, p.r, row * p.ld_r, t, cols);
        if (p.dr != nullptr) fetch_row<DT, TPR, NV>(at + C::kArrayDy + C::kArray, p.dr, row * p.ld_dr, t, cols);
      }
      cp_async_commit();
    }
  };
  float dg[NV][8];
#pragma unroll
  for (int i = 0; i < NV; ++i)
#pragma unroll
    for (int j = 0; j < 8; ++j) dg[i][j] = 0.0f;
  const float inv_n = 1.0f / (float)cols;
  auto count = [&](int i) {
    const int left = cols - (t + TPR * i) * 8;
    return ASYNC ? (left > 0 ? 8 : 0) : max(0, min(8, left));
  };
  int64_t row = (int64_t)blockIdx.x * kRows + sub;
#pragma unroll
  for (int d = 0; d < D - 1; ++d) fetch(row + d * step, d);
  int slot = 0;
  for (; row < p.rows; row += step) {
    const float rstd = p.rstd[row];
    if constexpr (ASYNC) {
      fetch(row + (D - 1) * step, slot == 0 ? D - 1 : slot - 1);
      cp_async_wait<D - 1>();
    }
    const char* at = mine + slot * C::kSlot;
    const char* dy_row = static_cast<const char*>(p.dy) + row * p.ld_dy * EY;
    const char* r_row = static_cast<const char*>(p.r) + row * p.ld_r * ES;
    const char* dr_row = static_cast<const char*>(p.dr) + row * p.ld_dr * ES;
    char* dx_row = static_cast<char*>(p.dx) + row * p.ld_dx * ES;
    float gdy[NV][8], xh[NV][8], u[NV][8];
    float s = 0.0f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c0 = (t + TPR * i) * 8;
      const int n = count(i);
      float gm[8];
      load8(p.gamma, p.gamma_dt, c0, n, p.vec_g && n == 8, gm);     // in L1 after the first row
      chunk8<DY, TPR, ASYNC>(at, i, dy_row, c0, n, p.vec_dy, gdy[i]);
      chunk8<DT, TPR, ASYNC>(at + C::kArrayDy, i, r_row, c0, n, p.vec_r, xh[i]);
      // without buffers the stream's gradient is loaded ahead of the row's sum
      if (!ASYNC && p.dr != nullptr) load8<DT>(dr_row, c0, n, p.vec_dr && n == 8, u[i]);
      float s0 = 0.0f, s1 = 0.0f;
#pragma unroll
      for (int j = 0; j < 8; j += 2) {
        mul2(xh[i][j], xh[i][j + 1], rstd, rstd, xh[i][j], xh[i][j + 1]);
        fma2(gdy[i][j], gdy[i][j + 1], xh[i][j], xh[i][j + 1], dg[i][j], dg[i][j + 1], dg[i][j], dg[i][j + 1]);
        mul2(gdy[i][j], gdy[i][j + 1], gm[j], gm[j + 1], gdy[i][j], gdy[i][j + 1]);
        fma2(gdy[i][j], gdy[i][j + 1], xh[i][j], xh[i][j + 1], s0, s1, s0, s1);
      }
      s += s0 + s1;
    }
    const float c = -row_sum<TPR>(s, s_red) * inv_n;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c0 = (t + TPR * i) * 8;
      const int n = count(i);
      float o[8];
#pragma unroll
      for (int j = 0; j < 8; j += 2) {
        fma2(xh[i][j], xh[i][j + 1], c, c, gdy[i][j], gdy[i][j + 1], o[j], o[j + 1]);
        mul2(o[j], o[j + 1], rstd, rstd, o[j], o[j + 1]);
      }
      if (p.dr != nullptr) {
        if constexpr (ASYNC) chunk8<DT, TPR, ASYNC>(at + C::kArrayDy + C::kArray, i, dr_row, c0, n, p.vec_dr, u[i]);
#pragma unroll
        for (int j = 0; j < 8; ++j) o[j] += u[i][j];
      }
      if (n > 0) store8<DT>(dx_row, c0, n, p.vec_dx && n == 8, o);
    }
    if constexpr (ASYNC) slot = slot + 1 == D ? 0 : slot + 1;
  }
  if constexpr (ASYNC) cp_async_wait<0>();
  float* s_dg = reinterpret_cast<float*>(s_rows + (ASYNC ? D * C::kSlot : 0));
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

// CTAs per SM: as many as the threads and the row buffers allow.
int64_t norm_per_sm(int threads, int smem, int most) {
  return std::max<int64_t>(1, std::min<int64_t>(std::min(2048 / threads, most), 220 * 1024 / (smem + 1024)));
}

template <int DT, int TPR, int NV, bool QUANT, bool ASYNC>
int launch_norm_k(const NormArgs& a, cudaStream_t s) {
  using C = NormCfg<DT, TPR, NV>;
  constexpr int kSmem = ASYNC ? C::kDepth * C::kSlot : 0;
  static unsigned long long attr = 0;
  if (int st = allow_smem(rmsnorm_kernel<DT, TPR, NV, QUANT, ASYNC>, kSmem, &attr)) return st;
  // at most 1024 threads' worth of registers (64 each)
  const int64_t most = norm_per_sm(C::kThreads, kSmem, 1024 / C::kThreads) * num_sms();
  const int64_t all = (a.rows + C::kRows - 1) / C::kRows;
  const int64_t grid = ASYNC ? std::min<int64_t>(all, most) : all;
  return launch_kernel(rmsnorm_kernel<DT, TPR, NV, QUANT, ASYNC>, dim3((unsigned)grid), dim3(C::kThreads), kSmem, s, 1,
                       a) == cudaSuccess ? APA_OK : APA_ERR_CUDA;
}

template <int DT, int TPR, int NV>
int launch_norm(const NormArgs& a, cudaStream_t s) {
  if constexpr (TPR > 32 && NormCfg<DT, TPR, NV>::kDepth >= 2) {
    if (a.vec_x && (!a.res || a.vec_res) && a.cols % 8 == 0)
      return a.q ? launch_norm_k<DT, TPR, NV, true, true>(a, s) : launch_norm_k<DT, TPR, NV, false, true>(a, s);
  }
  return a.q ? launch_norm_k<DT, TPR, NV, true, false>(a, s) : launch_norm_k<DT, TPR, NV, false, false>(a, s);
}

// Threads per row and chunks per thread: a warp per row up to 1024 columns (no
// block-wide sum), then 128 to 1024 threads with two chunks at most (four past
// 16384 columns), so that a row stays in registers. A warp per row against 128
// threads with rows fetched ahead, between 513 and 1024 columns (us): fp32 8192
// x 1024 13.2 and 18.0, with residual 23.1 and 35.5; bf16 8192 x 640 7.5 and
// 9.3, with residual 12.1 and 11.1; 8192 x 1024 9.2 and 9.5, with residual 14.4
// and 11.7, to E4M3 15.8 and 14.1; 33280 x 1024 36.9 and 27.5; 64 x 1024 3.1 and
// 1.6. fp32 rows and short 16-bit ones gain by it; 16-bit rows with a residual,
// and few or very many of them, lose.
template <int DT>
int norm_forward(const NormArgs& a, cudaStream_t s) {
  const int64_t chunks = (a.cols + 7) / 8;
  if (chunks <= 32) return launch_norm<DT, 32, 1>(a, s);
  if (chunks <= 64) return launch_norm<DT, 32, 2>(a, s);
  if (chunks <= 128) return launch_norm<DT, 32, 4>(a, s);
  if (chunks <= 256) return launch_norm<DT, 128, 2>(a, s);
  if (chunks <= 512) return launch_norm<DT, 256, 2>(a, s);
  if (chunks <= 1024) return launch_norm<DT, 512, 2>(a, s);
  if (chunks <= 2048) return launch_norm<DT, 1024, 2>(a, s);
  return launch_norm<DT, 1024, 4>(a, s);
}

// CTAs (= dgamma partial rows) of the backward: as many as are resident. A warp
// has a row up to 512 columns: past that the sums of dgamma would not leave a
// thread its registers.
int64_t norm_bwd_parts(int64_t rows, int64_t cols) {
  const int64_t chunks = (cols + 7) / 8;
  const int tpr = chunks <= 64 ? 32 : chunks <= 256 ? 128 : chunks <= 512 ? 256 : chunks <= 1024 ? 512 : 1024;
  const int per_cta = tpr < 128 ? 128 / tpr : 1;
  const int64_t per_sm = norm_bwd_resident(tpr, chunks <= 32 || (chunks > 64 && chunks <= 128) ? 1 : 2);
  return std::min<int64_t>((rows + per_cta - 1) / per_cta, per_sm * num_sms());
}

template <int DT, int DY, int TPR, int NV, bool ASYNC>
int launch_norm_bwd_k(const NormBwdArgs& a, int64_t parts, cudaStream_t s) {
  using C = NormBwdCfg<DT, DY, TPR, NV>;
  constexpr int kSmem = (ASYNC ? C::kDepth * C::kSlot : 0) + C::kSums;
  static unsigned long long attr = 0;
  if (int st = allow_smem(rmsnorm_bwd_kernel<DT, DY, TPR, NV, ASYNC>, kSmem, &attr)) return st;
  return launch_kernel(rmsnorm_bwd_kernel<DT, DY, TPR, NV, ASYNC>, dim3((unsigned)parts), dim3(C::kThreads), kSmem, s,
                       1, a) == cudaSuccess ? APA_OK : APA_ERR_CUDA;
}

template <int DT, int DY, int TPR, int NV>
int launch_norm_bwd(const NormBwdArgs& a, int64_t parts, cudaStream_t s) {
  // Short rows need no buffers where enough warps fit an SM to hide their loads:
  // 33280 x 512 fp32 41 us against 59 with buffers, 8192 x 1024 bf16 18 against
  // 20; but 16384 x 384 bf16 15 with and 23 without, 8192 x 2048 33 and 41.
  constexpr bool kBuffers = TPR >= 256 || (NV == 2 && (TPR == 128 || (DT != APA_DT_F32 && DY != APA_DT_F32)));
  if constexpr (kBuffers && NormBwdCfg<DT, DY, TPR, NV>::kDepth >= 2) {
    if (a.vec_dy && a.vec_r && (!a.dr || a.vec_dr) && a.cols % 8 == 0)
      return launch_norm_bwd_k<DT, DY, TPR, NV, true>(a, parts, s);
  }
  return launch_norm_bwd_k<DT, DY, TPR, NV, false>(a, parts, s);
}

template <int DT, int DY>
int norm_backward(const NormBwdArgs& a, int64_t parts, cudaStream_t s) {
  const int64_t chunks = (a.cols + 7) / 8;
  if (chunks <= 32) return launch_norm_bwd<DT, DY, 32, 1>(a, parts, s);
  if (chunks <= 64) return launch_norm_bwd<DT, DY, 32, 2>(a, parts, s);
  if (chunks <= 128) return launch_norm_bwd<DT, DY, 128, 1>(a, parts, s);
  if (chunks <= 256) return launch_norm_bwd<DT, DY, 128, 2>(a, parts, s);
  if (chunks <= 512) return launch_norm_bwd<DT, DY, 256, 2>(a, parts, s);
  if (chunks <= 1024) return launch_norm_bwd<DT, DY, 512, 2>(a, parts, s);
  if (chunks <= 2048) return launch_norm_bwd<DT, DY, 1024, 2>(a, parts, s);
  return launch_norm_bwd<DT, DY, 1024, 4>(a, parts, s);
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
             stream_out && vec16(stream_out, ld_stream, es) ? 1 : 0, y && vec16(y, ld_y, es) ? 1 : 0,
             vec16(gamma, 8, 4) ? 1 : 0};
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (dtype == APA_DT_F32) return norm_forward<APA_DT_F32>(a, s);
  if (dtype == APA_DT_F16) return norm_forward<APA_DT_F16>(a, s);
  return norm_forward<APA_DT_BF16>(a, s);
}

extern "C" int apa_rmsnorm_bwd_workspace(int64_t rows, int64_t cols, int64_t* bytes_out) {
  using namespace apa::blk;
  if (!bytes_out) return APA_ERR_INVALID;
  if (int st = norm_dims(rows, cols)) return st;
  *bytes_out = norm_bwd_parts(rows, cols) * cols * 4;
  return APA_OK;
}

extern "C" int apa_rmsnorm_bwd(const void* dy, int dy_dtype, int64_t ld_dy, const void* r, int64_t ld_r,
                               const float* rstd, const void* gamma, int gamma_dtype, const void* dr, int64_t ld_dr,
                               void* dx, int64_t ld_dx, int dtype, int64_t rows, int64_t cols, void* dgamma,
                               void* workspace, int64_t workspace_bytes, void* stream) {
  using namespace apa::blk;
  if (!dy || !r || !rstd || !gamma || !dx || !dgamma || !workspace) return APA_ERR_INVALID;
  if (int st = norm_dims(rows, cols)) return st;
  const int es = elem_bytes(dtype);
  if (es == 0 || elem_bytes(gamma_dtype) == 0) return APA_ERR_UNSUPPORTED;
  if (dy_dtype != dtype && dy_dtype != APA_DT_F32) return APA_ERR_UNSUPPORTED;
  if (ld_dy < cols || ld_r < cols || ld_dx < cols || (dr && ld_dr < cols)) return APA_ERR_INVALID;
  if ((reinterpret_cast<uintptr_t>(workspace) & 15u) != 0) return APA_ERR_ALIGN;
  const int64_t parts = norm_bwd_parts(rows, cols);
  if (workspace_bytes < parts * cols * 4) return APA_ERR_INVALID;
  NormBwdArgs a{dy, ld_dy, r, ld_r, rstd, gamma, gamma_dtype, dr, ld_dr, dx, ld_dx, static_cast<float*>(workspace),
                rows, cols, vec16(dy, ld_dy, elem_bytes(dy_dtype)) ? 1 : 0, vec16(r, ld_r, es) ? 1 : 0,
                dr && vec16(dr, ld_dr, es) ? 1 : 0, vec16(dx, ld_dx, es) ? 1 : 0, vec16(gamma, 8, 4) ? 1 : 0};
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  int st;
  if (dtype == APA_DT_F32) st = norm_backward<APA_DT_F32, APA_DT_F32>(a, parts, s);
  else if (dtype == APA_DT_F16 && dy_dtype == dtype) st = norm_backward<APA_DT_F16, APA_DT_F16>(a, parts, s);
  else if (dtype == APA_DT_F16) st = norm_backward<APA_DT_F16, APA_DT_F32>(a, parts, s);
  else if (dy_dtype == dtype) st = norm_backward<APA_DT_BF16, APA_DT_BF16>(a, parts, s);
  else st = norm_backward<APA_DT_BF16, APA_DT_F32>(a, parts, s);
  if (st != APA_OK) return st;
  return launch_colsum(a.part, parts, cols, dgamma, gamma_dtype, s);
}
