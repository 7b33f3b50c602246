// C ABI of the training layer norm (tj_norm_train.cuh).
#include <algorithm>
#include <type_traits>

#include "tj.h"
#include "tj_host.h"
#include "tj_norm_train.cuh"

namespace {

using tj_host::fail;

bool aligned(const void* p, size_t a) { return (reinterpret_cast<uintptr_t>(p) & (a - 1)) == 0; }
size_t vec_bytes(int dtype) { return dtype == TJ_F32 ? 16 : (dtype == TJ_E4M3 ? 4 : 8); }

// Runs f.template operator()<WR, NI, VEC>() for the width d: 512 columns a
// step, two steps a warp, up to four warps a row.
template <typename F>
int by_width(int d, bool vec, F&& f) {
  if (vec) {
    if (d <= 512) return f.template operator()<1, 1, true>();
    if (d <= 1024) return f.template operator()<1, 2, true>();
    if (d <= 2048) return f.template operator()<2, 2, true>();
    return f.template operator()<4, 2, true>();
  }
  if (d <= 1024) return f.template operator()<1, 2, false>();
  return f.template operator()<4, 2, false>();
}

template <typename T, typename Y>
struct Fwd {
  const tj::NormFwdParams& p;
  cudaStream_t st;
  template <int WR, int NI, bool VEC>
  int operator()() const {
    constexpr int rows = tj::kNormWarps / WR;
    tj::norm_fwd_kernel<T, Y, WR, NI, VEC>
        <<<(unsigned)((p.rows + rows - 1) / rows), 32 * tj::kNormWarps, 0, st>>>(p);
    TJH_CUDA(cudaGetLastError());
    return TJ_OK;
  }
};

template <typename T>
int fwd_y(int y_dtype, const tj::NormFwdParams& p, bool vec, cudaStream_t st) {
  switch (y_dtype) {
    case TJ_F32: return by_width(p.d, vec, Fwd<T, float>{p, st});
    case TJ_F16: return by_width(p.d, vec, Fwd<T, __half>{p, st});
    case TJ_BF16: return by_width(p.d, vec, Fwd<T, __nv_bfloat16>{p, st});
    default: return by_width(p.d, vec, Fwd<T, uint8_t>{p, st});
  }
}

// Warps that share a row in the backward pass: 512 columns each.
int bwd_wr(int d) { return d <= 512 ? 1 : (d <= 1024 ? 2 : (d <= 2048 ? 4 : 8)); }

// CTAs of the backward pass: as many as run at once, at most one per row group.
int bwd_grid(long long rows, int d, int sms) {
  const int wr = bwd_wr(d), warps = tj::norm_bwd_warps(wr);
  const long long groups = warps / wr;
  return (int)std::max<long long>(1, std::min<long long>((rows + groups - 1) / groups, (long long)tj::norm_bwd_ctas(wr) * sms));
}

template <typename DY, typename X, bool X8, int WR>
int bwd_launch(const tj::NormBwdParams& p, bool vec, int sms, cudaStream_t st) {
  const int grid = bwd_grid(p.rows, p.d, sms);
  if (vec) tj::norm_bwd_kernel<DY, X, X8, WR, true><<<grid, 32 * tj::norm_bwd_warps(WR), 0, st>>>(p);
  else tj::norm_bwd_kernel<DY, X, X8, WR, false><<<grid, 32 * tj::norm_bwd_warps(WR), 0, st>>>(p);
  TJH_CUDA(cudaGetLastError());
  if (grid > 1) {
    tj::column_sum_kernel<<<(2 * p.d + 7) / 8, 1024, 0, st>>>(p.partial, grid, 2 * p.d, p.dgamma, p.dbeta, p.d);
    TJH_CUDA(cudaGetLastError());
  }
  return TJ_OK;
}
template <typename DY, typename X, bool X8>
int bwd_width(const tj::NormBwdParams& p, bool vec, int sms, cudaStream_t st) {
  switch (bwd_wr(p.d)) {
    case 1: return bwd_launch<DY, X, X8, 1>(p, vec, sms, st);
    case 2: return bwd_launch<DY, X, X8, 2>(p, vec, sms, st);
    case 4: return bwd_launch<DY, X, X8, 4>(p, vec, sms, st);
    default: return bwd_launch<DY, X, X8, 8>(p, vec, sms, st);
  }
}

template <typename DY>
int bwd_x(int dx_dtype, bool x8, const tj::NormBwdParams& p, bool vec, int sms, cudaStream_t st) {
  switch (dx_dtype) {
    case TJ_F32: return x8 ? bwd_width<DY, float, true>(p, vec, sms, st) : bwd_width<DY, float, false>(p, vec, sms, st);
    case TJ_F16: return x8 ? bwd_width<DY, __half, true>(p, vec, sms, st) : bwd_width<DY, __half, false>(p, vec, sms, st);
    default:
      return x8 ? bwd_width<DY, __nv_bfloat16, true>(p, vec, sms, st)
                : bwd_width<DY, __nv_bfloat16, false>(p, vec, sms, st);
  }
}

int check_shape(long long rows, int d) {
  if (rows < 0 || d <= 0) return fail(TJ_ERR_INVALID, "rows %lld, width %d", rows, d);
  if (d > 4096) return fail(TJ_ERR_UNSUPPORTED, "LayerNorm width %d (need <= 4096)", d);
  if (rows > 0x7fffffffLL) return fail(TJ_ERR_UNSUPPORTED, "too many rows");
  return TJ_OK;
}
bool plain(int dtype) { return dtype == TJ_F32 || dtype == TJ_F16 || dtype == TJ_BF16; }

}  // namespace

extern "C" {

int tj_layernorm_train(const void* x, int x_dtype, const float* gamma, const float* beta, long long rows, int d,
                       float eps, const uint8_t* mask, void* y, int y_dtype, uint8_t* y_scales, float* mean,
                       float* rstd, void* x8_codes, uint8_t* x8_scales, void* stream) {
  TJH_CHECK(check_shape(rows, d));
  if (!plain(x_dtype) || !(plain(y_dtype) || y_dtype == TJ_E4M3)) return fail(TJ_ERR_INVALID, "unknown dtype");
  if (rows == 0) return TJ_OK;
  if (!x || !gamma || !beta || !y || !mean || !rstd) return fail(TJ_ERR_INVALID, "null argument");
  if ((y_dtype == TJ_E4M3) != (y_scales != nullptr) || (x8_codes == nullptr) != (x8_scales == nullptr))
    return fail(TJ_ERR_INVALID, "an 8-bit tensor needs its codes and its scales");
  int dev, sms;
  TJH_CHECK(tj_host::device(&dev, &sms));
  tj::NormFwdParams p{x, gamma, beta, mask, y, y_scales, mean, rstd, static_cast<uint8_t*>(x8_codes), x8_scales, rows, d, eps};
  const bool vec = d % 4 == 0 && aligned(x, vec_bytes(x_dtype)) && aligned(y, vec_bytes(y_dtype)) &&
                   aligned(gamma, 16) && aligned(beta, 16) && aligned(x8_codes, 4);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  switch (x_dtype) {
    case TJ_F32: return fwd_y<float>(y_dtype, p, vec, st);
    case TJ_F16: return fwd_y<__half>(y_dtype, p, vec, st);
    default: return fwd_y<__nv_bfloat16>(y_dtype, p, vec, st);
  }
}

int tj_layernorm_backward_workspace_bytes(long long rows, int d, size_t* bytes) {
  TJH_CHECK(check_shape(rows, d));
  if (!bytes) return fail(TJ_ERR_INVALID, "null argument");
  int dev, sms;
  TJH_CHECK(tj_host::device(&dev, &sms));
  const int grid = bwd_grid(rows, d, sms);
  *bytes = grid > 1 ? (size_t)grid * 2 * d * sizeof(float) : 0;
  return TJ_OK;
}

int tj_layernorm_backward(const void* dy, int dy_dtype, const void* x, const uint8_t* x8_scales, const float* gamma,
                          const float* mean, const float* rstd, long long rows, int d, const uint8_t* mask,
                          const void* resid_grad, void* dx, int dx_dtype, float* dgamma, float* dbeta,
                          void* workspace, size_t workspace_bytes, void* stream) {
  TJH_CHECK(check_shape(rows, d));
  if (!plain(dy_dtype) || !plain(dx_dtype)) return fail(TJ_ERR_INVALID, "unknown dtype");
  if (!gamma || !dgamma || !dbeta || (rows > 0 && (!dy || !x || !mean || !rstd || !dx)))
    return fail(TJ_ERR_INVALID, "null argument");
  if (!aligned(workspace, 4)) return fail(TJ_ERR_INVALID, "workspace not 4-byte aligned");
  size_t need = 0;
  TJH_CHECK(tj_layernorm_backward_workspace_bytes(rows, d, &need));
  if (workspace_bytes < need || (need > 0 && !workspace))
    return fail(TJ_ERR_INVALID, "workspace of %zu bytes, needs %zu", workspace_bytes, need);
  int dev, sms;
  TJH_CHECK(tj_host::device(&dev, &sms));
  tj::NormBwdParams p{dy, x, x8_scales, gamma, mean, rstd, mask, resid_grad, dx, dgamma, dbeta,
                      static_cast<float*>(workspace), rows, d};
  const bool x8 = x8_scales != nullptr;
  const bool vec = d % 4 == 0 && aligned(dy, vec_bytes(dy_dtype)) && aligned(x, vec_bytes(x8 ? TJ_E4M3 : dx_dtype)) &&
                   aligned(gamma, 16) && aligned(resid_grad, vec_bytes(dx_dtype)) && aligned(dx, vec_bytes(dx_dtype));
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  switch (dy_dtype) {
    case TJ_F32: return bwd_x<float>(dx_dtype, x8, p, vec, sms, st);
    case TJ_F16: return bwd_x<__half>(dx_dtype, x8, p, vec, sms, st);
    default: return bwd_x<__nv_bfloat16>(dx_dtype, x8, p, vec, sms, st);
  }
}

}  // extern "C"
