// A block-scaled linear layer's forward and backward as one call each: the
// casts, the norm in front, the products and the bias gradient are queued
// together, with every temporary in buffers of the caller. At a few
// microseconds per launch from C against several times that from an
// interpreter (argument checks, allocations, one foreign call each), this is
// what bounds small layers. The kernels are those of block_cast.cu, rmsnorm.cu
// and block_gemm.cu, called through their entry points, with their checks.
#include "block_scale.cuh"

namespace apa {
namespace blk {

int64_t pitch16(int64_t cols) { return (cols + 15) / 16 * 16; }
int64_t round256(int64_t n) { return (n + 255) / 256 * 256; }

int64_t scale_bytes(int64_t rows, int64_t cols) { return (cols + 511) / 512 * rows_padded(rows) * 4; }

// A packed block tensor: codes with the pitch pitch16(cols), then the scales.
int64_t packed_bytes(int64_t rows, int64_t cols) { return rows * pitch16(cols) + scale_bytes(rows, cols); }

struct Packed {
  uint8_t* q;
  int64_t ld;
  uint8_t* sc;
  Packed(const void* base, int64_t rows, int64_t cols)
      : q(static_cast<uint8_t*>(const_cast<void*>(base))), ld(pitch16(cols)), sc(q ? q + rows * ld : nullptr) {}
};

// Workspaces, in the order they are used.
struct FwdSpace { int64_t xq, wq, gemm, gemm_bytes, total; };
struct BwdSpace {
  int64_t dyq, dyt, xt, sums, dh, norm, gemm, norm_bytes, gemm_bytes, total;
  int split;             // units per tile of the first of both products
  bool dw_first;
};

// A few tokens through a kept weight: the product casts them itself.
bool casts_itself(int64_t M, int64_t N, int64_t K, int flags, bool aligned) {
  if (flags != 0 || M > 16) return false;
  const BlockPlan p = block_plan(M, N, K, aligned);
  return p.kind == 0 && p.bn == 16 && p.swap;
}

// flags: 1 the weight is cast, 2 a norm in front, 4 the transposed cast of x too
int fwd_space(int64_t M, int64_t N, int64_t K, int flags, int y_dtype, FwdSpace* s) {
  int64_t at = 0;
  auto take = [&](int64_t bytes) {
    const int64_t here = at;
    at += round256(bytes);
    return here;
  };
  // whether y's rows are aligned is known only in the call: room for both
  const bool itself = casts_itself(M, N, K, flags, true) && casts_itself(M, N, K, flags, false);
  s->xq = take(itself ? 0 : packed_bytes(M, K));
  s->wq = take((flags & 1) ? packed_bytes(N, K) : 0);
  s->gemm_bytes = 0;
  if (!itself)
    if (int st = apa_block_gemm_workspace(M, N, K, y_dtype, APA_BLOCK_AUTO, &s->gemm_bytes)) return st;
  s->gemm = take(s->gemm_bytes);
  s->total = at;
  return APA_OK;
}

enum { kWantDx = 1, kWantDw = 2, kWantDb = 4, kNorm = 8 };

int bwd_space(int64_t M, int64_t N, int64_t K, int flags, int dtype, int dw_dtype, BwdSpace* s) {
  int64_t at = 0;
  auto take = [&](int64_t bytes) {
    const int64_t here = at;
    at += round256(bytes);
    return here;
  };
  const bool dx = flags & kWantDx, dw = flags & kWantDw, norm = flags & kNorm;
  s->dyq = take(dx || !dw ? packed_bytes(M, N) : 0);     // a cast that only sums columns writes its rows form
  s->dyt = take(dw ? packed_bytes(N, M) : 0);
  s->xt = take(dw && norm ? packed_bytes(K, M) : 0);
  s->sums = take((flags & kWantDb) ? (M + 127) / 128 * N * 4 : 0);
  s->dh = take(dx && norm ? M * K * 4 : 0);
  s->norm_bytes = 0;
  if (dx && norm)
    if (int st = apa_rmsnorm_bwd_workspace(M, K, &s->norm_bytes)) return st;
  s->norm = take(s->norm_bytes);
  s->split = 1;
  s->gemm_bytes = 0;
  if (dw && dx) {
    // both products in one launch, the one with the longer tiles first
    OutArgs ow{}, ox{};
    ow.M = (int)N; ow.N = (int)K; ow.out_dt = dw_dtype;
    ox.M = (int)M; ox.N = (int)K; ox.out_dt = norm ? APA_DT_F32 : dtype;
    s->dw_first = M >= N;
    s->split = s->dw_first ? dual_split(ow, M, ox, N) : dual_split(ox, N, ow, M);
    s->gemm_bytes = s->dw_first ? split_bytes(N, K, s->split) : split_bytes(M, K, s->split);
  } else if (dw) {
    if (int st = apa_block_gemm_workspace(N, K, M, dw_dtype, APA_BLOCK_AUTO, &s->gemm_bytes)) return st;
  } else if (dx) {
    const int dt = norm ? APA_DT_F32 : dtype;
    if (int st = apa_block_gemm_workspace(M, K, N, dt, APA_BLOCK_AUTO, &s->gemm_bytes)) return st;
  }
  s->gemm = take(s->gemm_bytes);
  s->total = at;
  return APA_OK;
}

int layer_dims(int64_t M, int64_t N, int64_t K) {
  const int64_t top = (1ll << 31) - 256;
  return M <= 0 || N <= 0 || K <= 0 || M > top || N > top || K > top ? APA_ERR_INVALID : APA_OK;
}

bool aligned_16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

}  // namespace blk
}  // namespace apa

extern "C" int apa_block_linear_fwd_workspace(int64_t M, int64_t N, int64_t K, int flags, int y_dtype,
                                              int64_t* bytes_out) {
  using namespace apa::blk;
  if (!bytes_out || (flags & ~7) != 0) return APA_ERR_INVALID;
  if (int st = layer_dims(M, N, K)) return st;
  if (elem_bytes(y_dtype) == 0) return APA_ERR_UNSUPPORTED;
  FwdSpace s;
  if (int st = fwd_space(M, N, K, flags, y_dtype, &s)) return st;
  *bytes_out = s.total;
  return APA_OK;
}

extern "C" int apa_block_linear_fwd(const void* x, int x_dtype, int64_t ld_x, const void* residual, int64_t ld_res,
                                    const void* gamma, int gamma_dtype, float eps, void* stream_out, int64_t ld_stream,
                                    float* rstd, void* xt, const void* w, int w_dtype, int64_t ld_w, const void* wq,
                                    void* wt, const void* bias, int bias_dtype, void* y, int y_dtype, int64_t ld_y,
                                    int64_t M, int64_t N, int64_t K, void* workspace, int64_t workspace_bytes,
                                    void* stream) {
  using namespace apa::blk;
  if (int st = layer_dims(M, N, K)) return st;
  if (!x || !y || (w == nullptr) == (wq == nullptr)) return APA_ERR_INVALID;
  if (!gamma && (residual || stream_out || rstd)) return APA_ERR_INVALID;
  if ((gamma && xt) || (!w && wt)) return APA_ERR_INVALID;
  if (!aligned_16(workspace) || !aligned_16(xt) || !aligned_16(wq) || !aligned_16(wt)) return APA_ERR_ALIGN;
  // all refusals come before the first launch
  const int es = elem_bytes(y_dtype);
  if (elem_bytes(x_dtype) == 0 || es == 0 || (w && elem_bytes(w_dtype) == 0) || (bias && elem_bytes(bias_dtype) == 0) ||
      (gamma && elem_bytes(gamma_dtype) == 0))
    return APA_ERR_UNSUPPORTED;
  if (ld_x < K || (w && ld_w < K) || ld_y < N) return APA_ERR_INVALID;
  const int flags = (w ? 1 : 0) | (gamma ? 2 : 0) | (xt ? 4 : 0);
  FwdSpace f;
  if (int st = fwd_space(M, N, K, flags, y_dtype, &f)) return st;
  if (workspace_bytes < f.total || (f.total > 0 && !workspace)) return APA_ERR_INVALID;
  char* ws = static_cast<char*>(workspace);
  const OutArgs o{y, ld_y, y_dtype, bias, bias_dtype, 0, vec16(y, ld_y, es) ? 1 : 0, (int)M, (int)N};
  if (casts_itself(M, N, K, flags, o.vec && (N * es) % 16 == 0)) {
    const Packed W(wq, N, K);
    return small_linear(x, x_dtype, ld_x, Operand{W.q, W.ld, W.sc, N}, K, o, static_cast<cudaStream_t>(stream));
  }
  const Packed X(ws + f.xq, M, K), XT(xt, K, M), W(w ? ws + f.wq : wq, N, K), WT(wt, K, N);
  int st;
  if (gamma || !w) {
    if (gamma)
      st = apa_rmsnorm_fwd(x, ld_x, residual, ld_res, gamma, gamma_dtype, x_dtype, M, K, eps, stream_out, ld_stream,
                           nullptr, 0, X.q, X.ld, X.sc, rstd, stream);
    else
      st = apa_block_cast(x, x_dtype, M, K, ld_x, nullptr, nullptr, 0, 0, X.q, X.ld, X.sc, nullptr, 0, nullptr, nullptr,
                          stream);
    if (!st && w)
      st = apa_block_cast(w, w_dtype, N, K, ld_w, nullptr, nullptr, 0, 1, W.q, W.ld, W.sc, WT.q, WT.ld, WT.sc, nullptr,
                          stream);
  } else {
    const CastArgs cw = cast_args(w, elem_bytes(w_dtype), N, K, ld_w, nullptr, nullptr, 0, W.q, W.ld, W.sc, WT.q,
                                  WT.ld, WT.sc, nullptr);
    const CastArgs cx = cast_args(x, elem_bytes(x_dtype), M, K, ld_x, nullptr, nullptr, 0, X.q, X.ld, X.sc, XT.q,
                                  XT.ld, XT.sc, nullptr);
    st = cast_pair(cw, w_dtype, cx, x_dtype, static_cast<cudaStream_t>(stream));
  }
  if (st) return st;
  return apa_block_gemm(X.q, X.ld, X.sc, W.q, W.ld, W.sc, bias, bias_dtype, y, y_dtype, ld_y, M, N, K, 0,
                        APA_BLOCK_AUTO, ws + f.gemm, f.gemm_bytes, stream);
}

extern "C" int apa_block_linear_bwd_workspace(int64_t M, int64_t N, int64_t K, int flags, int dtype, int dw_dtype,
                                              int64_t* bytes_out) {
  using namespace apa::blk;
  if (!bytes_out || (flags & ~15) != 0) return APA_ERR_INVALID;
  if (int st = layer_dims(M, N, K)) return st;
  if (elem_bytes(dtype) == 0 || elem_bytes(dw_dtype) == 0) return APA_ERR_UNSUPPORTED;
  BwdSpace s;
  if (int st = bwd_space(M, N, K, flags, dtype, dw_dtype, &s)) return st;
  *bytes_out = s.total;
  return APA_OK;
}

extern "C" int apa_block_linear_bwd(const void* dy, int dy_dtype, int64_t ld_dy, const void* wt, const void* xt,
                                    const void* r, int64_t ld_r, const float* rstd, const void* gamma, int gamma_dtype,
                                    const void* dr, int64_t ld_dr, void* dx, int dtype, int64_t ld_dx, void* dgamma,
                                    void* dw, int dw_dtype, int64_t ld_dw, void* db, int db_dtype, int64_t M, int64_t N,
                                    int64_t K, void* workspace, int64_t workspace_bytes, void* stream) {
  using namespace apa::blk;
  if (int st = layer_dims(M, N, K)) return st;
  const bool norm = gamma != nullptr;
  if (!dy || !workspace || (!dx && !dw && !db) || ld_dy < N) return APA_ERR_INVALID;
  if (norm && (!r || !rstd || ld_r < K || (dx != nullptr) != (dgamma != nullptr))) return APA_ERR_INVALID;
  if (!norm && (r || rstd || dgamma || dr)) return APA_ERR_INVALID;
  if ((dx && (!wt || ld_dx < K)) || (dw && (ld_dw < K || (!norm && !xt)))) return APA_ERR_INVALID;
  if (dr && ld_dr < K) return APA_ERR_INVALID;
  if (elem_bytes(dy_dtype) == 0 || elem_bytes(dtype) == 0 || (dw && elem_bytes(dw_dtype) == 0) ||
      (db && elem_bytes(db_dtype) == 0) || (norm && elem_bytes(gamma_dtype) == 0))
    return APA_ERR_UNSUPPORTED;
  if (!aligned_16(workspace) || !aligned_16(wt) || !aligned_16(xt)) return APA_ERR_ALIGN;
  const int flags = (dx ? kWantDx : 0) | (dw ? kWantDw : 0) | (db ? kWantDb : 0) | (norm ? kNorm : 0);
  BwdSpace s;
  if (int st = bwd_space(M, N, K, flags, dtype, dw ? dw_dtype : APA_DT_F32, &s)) return st;
  if (workspace_bytes < s.total) return APA_ERR_INVALID;
  char* ws = static_cast<char*>(workspace);
  const bool rows_form = dx || !dw;
  const Packed DY(rows_form ? ws + s.dyq : nullptr, M, N), DYT(dw ? ws + s.dyt : nullptr, N, M), WT(wt, K, N);
  float* sums = db ? reinterpret_cast<float*>(ws + s.sums) : nullptr;
  int st = apa_block_cast(dy, dy_dtype, M, N, ld_dy, nullptr, nullptr, 0, 0, DY.q, DY.ld, DY.sc, DYT.q, DYT.ld, DYT.sc,
                          sums, stream);
  if (st) return st;
  // with both products to come, their launch adds the column sums
  const bool both = dw && dx;
  const int64_t parts = (M + 127) / 128;
  const bool later = db && both && dual_adds(parts, s.dw_first ? M : N, s.split);
  if (db && !later) {
    st = apa_block_colsum(sums, parts, N, db, db_dtype, stream);
    if (st) return st;
  }
  const Packed XT(norm ? ws + s.xt : xt, K, M);
  if (dw && norm) {
    // the norm's output again, from the stream, with scales along the tokens
    st = apa_block_cast(r, dtype, M, K, ld_r, rstd, gamma, gamma_dtype, 0, nullptr, 0, nullptr, XT.q, XT.ld, XT.sc,
                        nullptr, stream);
    if (st) return st;
  }
  // behind a norm the gradient of its output stays in fp32: rounding it would
  // add to the rounding of dx and of dgamma's terms
  void* dh = norm ? static_cast<void*>(ws + s.dh) : dx;
  const int dh_dtype = norm ? APA_DT_F32 : dtype;
  const int64_t ld_dh = norm ? K : ld_dx;
  if (both) {
    auto out = [](void* p, int dt, int64_t ld, int64_t rows, int64_t cols) {
      return OutArgs{p, ld, dt, nullptr, 0, 0, vec16(p, ld, elem_bytes(dt)) ? 1 : 0, (int)rows, (int)cols};
    };
    const Operand gw{DYT.q, DYT.ld, DYT.sc, N}, xw{XT.q, XT.ld, XT.sc, K};
    const Operand gx{DY.q, DY.ld, DY.sc, M}, wx{WT.q, WT.ld, WT.sc, K};
    const OutArgs ow = out(dw, dw_dtype, ld_dw, N, K), ox = out(dh, dh_dtype, ld_dh, M, K);
    const ColumnSums sum = later ? ColumnSums{sums, (int)parts, (int)N, db, db_dtype} : ColumnSums{};
    cudaStream_t cs = static_cast<cudaStream_t>(stream);
    st = s.dw_first ? block_gemm_dual(gw, xw, M, ow, gx, wx, N, ox, sum, s.split, ws + s.gemm, cs)
                    : block_gemm_dual(gx, wx, N, ox, gw, xw, M, ow, sum, s.split, ws + s.gemm, cs);
  } else if (dw) {
    st = apa_block_gemm(DYT.q, DYT.ld, DYT.sc, XT.q, XT.ld, XT.sc, nullptr, 0, dw, dw_dtype, ld_dw, N, K, M, 0,
                        APA_BLOCK_AUTO, ws + s.gemm, s.gemm_bytes, stream);
  } else if (dx) {
    st = apa_block_gemm(DY.q, DY.ld, DY.sc, WT.q, WT.ld, WT.sc, nullptr, 0, dh, dh_dtype, ld_dh, M, K, N, 0,
                        APA_BLOCK_AUTO, ws + s.gemm, s.gemm_bytes, stream);
  }
  if (st || !dx || !norm) return st;
  st = apa_rmsnorm_bwd(dh, APA_DT_F32, K, r, ld_r, rstd, gamma, gamma_dtype, dr, ld_dr, dx, ld_dx, dtype, M, K, dgamma,
                       ws + s.norm, s.norm_bytes, stream);
  return st;
}
