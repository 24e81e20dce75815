// Layer norm and dropout: the C entries (checks of arguments, workspace size) in front of the kernels in norm_kernels.h.
#include "norm.h"

namespace {

// sizes the kernels' index arithmetic holds for: M F elements counted in int64, columns in int32
constexpr int64_t MAX_F = 1 << 24;
constexpr int64_t MAX_N = (int64_t)1 << 40;

bool bad_dtype(int d) { return d != GSAGE_F32 && d != GSAGE_BF16 && d != GSAGE_F16; }
// The mask counts the rate as the fp32 number that the projection's epilogue takes (so the masks are the same); the scale
// is that of the rate as given: 1 - p of a rounded p is off by up to 2^-25 / (1 - p).
bool bad_p(double p) { return !(p >= 0. && (float)p < 1.f); }
NormDrop drop_of(double p, uint64_t seed, const int64_t *seed_dev) { return {(float)p, (float)(1. / (1. - p)), seed, seed_dev}; }

}  // namespace

extern "C" int gsage_dropout(const void *x, int64_t n, int dtype, double p, uint64_t seed, const int64_t *seed_dev,
                             void *out, gsage_stream_t stream) {
  if (n < 0 || bad_dtype(dtype) || bad_p(p)) return GSAGE_ERR_INVALID_ARG;
  if (n == 0) return GSAGE_OK;
  if (!x || !out) return GSAGE_ERR_INVALID_ARG;
  if (n > MAX_N) return GSAGE_ERR_UNSUPPORTED;
  const auto go = dtype == GSAGE_F32 ? norm_dropout_f32 : dtype == GSAGE_BF16 ? norm_dropout_bf16 : norm_dropout_f16;
  return go(x, n, drop_of(p, seed, seed_dev), out, gs_stream(stream));
}

extern "C" int gsage_layer_norm_fwd(const void *x, const void *residual, const void *weight, const void *bias, int64_t M,
                                    int64_t F, int dtype, int wdtype, float eps, double p, uint64_t seed,
                                    const int64_t *seed_dev, void *y, void *sum, float *mean, float *rstd,
                                    gsage_stream_t stream) {
  if (M < 0 || F <= 0 || bad_dtype(dtype) || bad_p(p) || !(eps >= 0.f)) return GSAGE_ERR_INVALID_ARG;
  if (wdtype != dtype && wdtype != GSAGE_F32) return GSAGE_ERR_INVALID_ARG;
  if ((mean == nullptr) != (rstd == nullptr)) return GSAGE_ERR_INVALID_ARG;
  if (M == 0) return GSAGE_OK;
  if (!x || !y) return GSAGE_ERR_INVALID_ARG;
  if (F > MAX_F || M > MAX_N / F) return GSAGE_ERR_UNSUPPORTED;
  const auto go = dtype == GSAGE_F32 ? norm_fwd_f32 : dtype == GSAGE_BF16 ? norm_fwd_bf16 : norm_fwd_f16;
  return go(NormFwd{x, residual, weight, bias, M, F, wdtype, eps, drop_of(p, seed, seed_dev), y, sum, mean, rstd},
            gs_stream(stream));
}

static size_t ws_bytes_of(int64_t M, int64_t F, int dtype, bool join) {
  if (M < 0 || F <= 0 || F > MAX_F || M > MAX_N / F || bad_dtype(dtype)) return 0;
  return gs_align_up((size_t)norm_ws_floats(M, F, dtype == GSAGE_F32 ? 4 : 2, join) * sizeof(float), 256);
}
extern "C" size_t gsage_layer_norm_bwd_workspace_bytes(int64_t M, int64_t F, int dtype) { return ws_bytes_of(M, F, dtype, false); }
extern "C" size_t gsage_layer_norm_bwd_joined_workspace_bytes(int64_t M, int64_t F, int dtype) {
  return ws_bytes_of(M, F, dtype, true);
}

extern "C" int gsage_layer_norm_bwd(const void *grad_y, const void *grad_sum, const void *x, const void *residual,
                                    const void *weight, const float *mean, const float *rstd, int64_t M, int64_t F,
                                    int dtype, int wdtype, double p, uint64_t seed, const int64_t *seed_dev, void *grad_x,
                                    void *grad_residual, void *grad_weight, void *grad_bias, void *ws, size_t ws_bytes,
                                    gsage_stream_t stream) {
  if (M < 0 || F <= 0 || bad_dtype(dtype) || bad_p(p)) return GSAGE_ERR_INVALID_ARG;
  if (wdtype != dtype && wdtype != GSAGE_F32) return GSAGE_ERR_INVALID_ARG;
  if (F > MAX_F || M > MAX_N / F) return GSAGE_ERR_UNSUPPORTED;
  if (M > 0 && (!grad_y || !x || !mean || !rstd)) return GSAGE_ERR_INVALID_ARG;
  const NormBwd n{grad_y, grad_sum, x, residual, weight, mean, rstd, M, F, wdtype, drop_of(p, seed, seed_dev),
                  grad_x, grad_residual, grad_weight, grad_bias, (float *)ws};
  if (grad_weight || grad_bias) {
    if (!ws) return GSAGE_ERR_INVALID_ARG;
    if (ws_bytes < ws_bytes_of(M, F, dtype, n.joined())) return GSAGE_ERR_WORKSPACE;
  }
  const auto go = dtype == GSAGE_F32 ? norm_bwd_f32 : dtype == GSAGE_BF16 ? norm_bwd_bf16 : norm_bwd_f16;
  return go(n, gs_stream(stream));
}
