// Layer norm and counter-based dropout, forward and backward, and the two joined with a residual sum.
//
//   z = residual + dropout(x);  y = (z - mean) rstd w + b
//   a = g w;  h = (z - mean) rstd;  dz = rstd (a - mean(a) - h mean(a h)) + grad_sum
//   grad_residual = dz;  grad_x = dropout'(dz);  grad_w = sum_rows g h;  grad_b = sum_rows g
//
// Neither the mask nor z is stored: both are formed again from (seed, index) and from x and residual.
#include "gsage_common.h"
#include "gsage_dropout.h"

namespace {

__device__ __forceinline__ float to_f(float v) { return v; }
__device__ __forceinline__ float to_f(__bf16 v) { return (float)v; }
__device__ __forceinline__ float to_f(_Float16 v) { return (float)v; }

struct Drop {              // p = 0: no mask
  float p, inv_keep;
  uint64_t seed;
  const int64_t *seed_dev;
  __device__ __forceinline__ uint64_t key() const { return seed_dev ? (uint64_t)*seed_dev : seed; }
};

__device__ __forceinline__ float drop1(float v, int64_t idx, uint64_t key, const Drop &d) {
  if (d.p <= 0.f) return v;
  return dropout_keep(key, (uint64_t)idx, d.p) ? v * d.inv_keep : 0.f;
}

template <typename T>
__global__ void __launch_bounds__(256) dropout_k(const T *x, int64_t n, Drop d, T *out) {
  const uint64_t key = d.key();
  const int64_t stride = (int64_t)gridDim.x * 256;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += stride)
    out[i] = (T)drop1(to_f(x[i]), i, key, d);
}

// sum over the 256 threads of a workgroup, in every thread
__device__ __forceinline__ float block_sum(float v) {
  __shared__ float part[4];
  v = gs_wave_sum(v);
  __syncthreads();
  if (gs_lane() == 0) part[threadIdx.x >> 6] = v;
  __syncthreads();
  return part[0] + part[1] + part[2] + part[3];
}

__device__ __forceinline__ float load_w(const void *w, int wdtype, int64_t c) {
  if (wdtype == GSAGE_F32) return ((const float *)w)[c];
  if (wdtype == GSAGE_BF16) return (float)((const __bf16 *)w)[c];
  return (float)((const _Float16 *)w)[c];
}
__device__ __forceinline__ void store_w(void *w, int wdtype, int64_t c, float v) {
  if (wdtype == GSAGE_F32) ((float *)w)[c] = v;
  else if (wdtype == GSAGE_BF16) ((__bf16 *)w)[c] = (__bf16)v;
  else ((_Float16 *)w)[c] = (_Float16)v;
}

template <typename T> struct Ln {
  const T *x, *res;
  const void *w, *b;
  int64_t M, F;
  int wdtype;
  Drop d;
  __device__ __forceinline__ float z(int64_t idx, uint64_t key) const {
    const float v = drop1(to_f(x[idx]), idx, key, d);
    return res ? to_f(res[idx]) + v : v;
  }
};

template <typename T>
__global__ void __launch_bounds__(256) ln_fwd_k(Ln<T> a, float eps, T *y, T *sum, float *mean, float *rstd) {
  const uint64_t key = a.d.key();
  const float inv_f = 1.0f / (float)a.F;
  for (int64_t r = blockIdx.x; r < a.M; r += gridDim.x) {
    const int64_t base = r * a.F;
    float s = 0.f, q = 0.f;
    for (int64_t c = threadIdx.x; c < a.F; c += 256) s += a.z(base + c, key);
    const float m = block_sum(s) * inv_f;
    for (int64_t c = threadIdx.x; c < a.F; c += 256) { const float t = a.z(base + c, key) - m; q += t * t; }
    const float rs = 1.0f / sqrtf(block_sum(q) * inv_f + eps);
    for (int64_t c = threadIdx.x; c < a.F; c += 256) {
      const float z = a.z(base + c, key);
      const float h = (z - m) * rs;
      const float w = a.w ? load_w(a.w, a.wdtype, c) : 1.f, b = a.b ? load_w(a.b, a.wdtype, c) : 0.f;
      y[base + c] = (T)(h * w + b);
      if (sum) sum[base + c] = (T)z;
    }
    if (mean && threadIdx.x == 0) { mean[r] = m; rstd[r] = rs; }
  }
}

template <typename T>
__global__ void __launch_bounds__(256) ln_dz_k(Ln<T> a, const T *g, const T *gsum, const float *mean,
                                               const float *rstd, T *gx, T *gres) {
  const uint64_t key = a.d.key();
  const float inv_f = 1.0f / (float)a.F;
  for (int64_t r = blockIdx.x; r < a.M; r += gridDim.x) {
    const int64_t base = r * a.F;
    const float m = mean[r], rs = rstd[r];
    float s1 = 0.f, s2 = 0.f;
    for (int64_t c = threadIdx.x; c < a.F; c += 256) {
      const float h = (a.z(base + c, key) - m) * rs;
      const float t = to_f(g[base + c]) * (a.w ? load_w(a.w, a.wdtype, c) : 1.f);
      s1 += t; s2 += t * h;
    }
    s1 = block_sum(s1) * inv_f;
    s2 = block_sum(s2) * inv_f;
    for (int64_t c = threadIdx.x; c < a.F; c += 256) {
      const int64_t i = base + c;
      const float h = (a.z(i, key) - m) * rs;
      const float t = to_f(g[i]) * (a.w ? load_w(a.w, a.wdtype, c) : 1.f);
      float dz = rs * (t - s1 - h * s2);
      if (gsum) dz += to_f(gsum[i]);
      if (gres) gres[i] = (T)dz;
      if (gx) gx[i] = (T)drop1(dz, i, key, a.d);
    }
  }
}

// grad_w / grad_b: slab s of workgroup (column tile, s) holds the sums over its rows
template <typename T>
__global__ void __launch_bounds__(256) ln_dw_k(Ln<T> a, const T *g, const float *mean, const float *rstd,
                                               float *ws) {
  const int64_t c = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (c >= a.F) return;
  const uint64_t key = a.d.key();
  float dw = 0.f, db = 0.f;
  for (int64_t r = blockIdx.y; r < a.M; r += gridDim.y) {
    const float gv = to_f(g[r * a.F + c]);
    dw += gv * ((a.z(r * a.F + c, key) - mean[r]) * rstd[r]);
    db += gv;
  }
  float *slab = ws + (int64_t)blockIdx.y * 2 * a.F;
  slab[c] = dw;
  slab[a.F + c] = db;
}

__global__ void __launch_bounds__(256) ln_dw_sum_k(const float *ws, int slabs, int64_t F, int wdtype, void *gw,
                                                   void *gb) {
  const int64_t c = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (c >= F) return;
  double dw = 0., db = 0.;
  for (int s = 0; s < slabs; ++s) {
    dw += ws[(int64_t)s * 2 * F + c];
    db += ws[(int64_t)s * 2 * F + F + c];
  }
  if (gw) store_w(gw, wdtype, c, (float)dw);
  if (gb) store_w(gb, wdtype, c, (float)db);
}

int ln_slabs(int64_t M) { return (int)(M < 256 ? M : 256); }

// sizes the kernels' index arithmetic holds for: M F elements counted in int64, columns in int32
constexpr int64_t MAX_F = 1 << 24;
constexpr int64_t MAX_N = (int64_t)1 << 40;

bool bad_dtype(int d) { return d != GSAGE_F32 && d != GSAGE_BF16 && d != GSAGE_F16; }
bool bad_p(float p) { return !(p >= 0.f && p < 1.f); }

template <typename T>
int ln_fwd(const void *x, const void *res, const void *w, const void *b, int64_t M, int64_t F, int wdtype, float eps,
           const Drop &d, void *y, void *sum, float *mean, float *rstd, hipStream_t st) {
  Ln<T> a{(const T *)x, (const T *)res, w, b, M, F, wdtype, d};
  hipLaunchKernelGGL(ln_fwd_k<T>, dim3(gs_grid(M, 1)), dim3(256), 0, st, a, eps, (T *)y, (T *)sum, mean, rstd);
  GSAGE_CHECK_LAUNCH();
  return GSAGE_OK;
}

template <typename T>
int ln_bwd(const void *g, const void *gsum, const void *x, const void *res, const void *w, const float *mean,
           const float *rstd, int64_t M, int64_t F, int wdtype, const Drop &d, void *gx, void *gres, void *gw, void *gb,
           float *ws, hipStream_t st) {
  Ln<T> a{(const T *)x, (const T *)res, w, nullptr, M, F, wdtype, d};
  const unsigned tiles = (unsigned)((F + 255) / 256);
  if (M > 0 && (gx || gres)) {
    hipLaunchKernelGGL(ln_dz_k<T>, dim3(gs_grid(M, 1)), dim3(256), 0, st, a, (const T *)g, (const T *)gsum, mean, rstd,
                       (T *)gx, (T *)gres);
    GSAGE_CHECK_LAUNCH();
  }
  if (gw || gb) {
    if (M > 0) {
      hipLaunchKernelGGL(ln_dw_k<T>, dim3(tiles, ln_slabs(M)), dim3(256), 0, st, a, (const T *)g, mean, rstd, ws);
      GSAGE_CHECK_LAUNCH();
    }
    hipLaunchKernelGGL(ln_dw_sum_k, dim3(tiles), dim3(256), 0, st, ws, ln_slabs(M), F, wdtype, gw, gb);
    GSAGE_CHECK_LAUNCH();
  }
  return GSAGE_OK;
}

}  // namespace

extern "C" int gsage_dropout(const void *x, int64_t n, int dtype, float p, uint64_t seed, const int64_t *seed_dev,
                             void *out, gsage_stream_t stream) {
  if (n < 0 || bad_dtype(dtype) || bad_p(p)) return GSAGE_ERR_INVALID_ARG;
  if (n == 0) return GSAGE_OK;
  if (!x || !out) return GSAGE_ERR_INVALID_ARG;
  if (n > MAX_N) return GSAGE_ERR_UNSUPPORTED;
  const Drop d{p, 1.0f / (1.0f - p), seed, seed_dev};
  const dim3 grid(gs_grid(n, 256)), block(256);
  hipStream_t st = gs_stream(stream);
  if (dtype == GSAGE_F32) hipLaunchKernelGGL(dropout_k<float>, grid, block, 0, st, (const float *)x, n, d, (float *)out);
  else if (dtype == GSAGE_BF16) hipLaunchKernelGGL(dropout_k<__bf16>, grid, block, 0, st, (const __bf16 *)x, n, d, (__bf16 *)out);
  else hipLaunchKernelGGL(dropout_k<_Float16>, grid, block, 0, st, (const _Float16 *)x, n, d, (_Float16 *)out);
  GSAGE_CHECK_LAUNCH();
  return GSAGE_OK;
}

extern "C" int gsage_layer_norm_fwd(const void *x, const void *residual, const void *weight, const void *bias, int64_t M,
                                    int64_t F, int dtype, int wdtype, float eps, float p, uint64_t seed,
                                    const int64_t *seed_dev, void *y, void *sum, float *mean, float *rstd,
                                    gsage_stream_t stream) {
  if (M < 0 || F <= 0 || bad_dtype(dtype) || bad_p(p) || !(eps >= 0.f)) return GSAGE_ERR_INVALID_ARG;
  if (wdtype != dtype && wdtype != GSAGE_F32) return GSAGE_ERR_INVALID_ARG;
  if ((mean == nullptr) != (rstd == nullptr)) return GSAGE_ERR_INVALID_ARG;
  if (M == 0) return GSAGE_OK;
  if (!x || !y) return GSAGE_ERR_INVALID_ARG;
  if (F > MAX_F || M > MAX_N / F) return GSAGE_ERR_UNSUPPORTED;
  const Drop d{p, 1.0f / (1.0f - p), seed, seed_dev};
  const auto go = dtype == GSAGE_F32 ? ln_fwd<float> : dtype == GSAGE_BF16 ? ln_fwd<__bf16> : ln_fwd<_Float16>;
  return go(x, residual, weight, bias, M, F, wdtype, eps, d, y, sum, mean, rstd, gs_stream(stream));
}

extern "C" size_t gsage_layer_norm_bwd_workspace_bytes(int64_t M, int64_t F, int dtype) {
  if (M < 0 || F <= 0 || F > MAX_F || bad_dtype(dtype)) return 0;
  const size_t slabs = (size_t)ln_slabs(M);
  return gs_align_up((slabs ? slabs : 1) * 2 * (size_t)F * sizeof(float), 256);
}

extern "C" int gsage_layer_norm_bwd(const void *grad_y, const void *grad_sum, const void *x, const void *residual,
                                    const void *weight, const float *mean, const float *rstd, int64_t M, int64_t F,
                                    int dtype, int wdtype, float p, uint64_t seed, const int64_t *seed_dev, void *grad_x,
                                    void *grad_residual, void *grad_weight, void *grad_bias, void *ws, size_t ws_bytes,
                                    gsage_stream_t stream) {
  if (M < 0 || F <= 0 || bad_dtype(dtype) || bad_p(p)) return GSAGE_ERR_INVALID_ARG;
  if (wdtype != dtype && wdtype != GSAGE_F32) return GSAGE_ERR_INVALID_ARG;
  if (F > MAX_F || M > MAX_N / F) return GSAGE_ERR_UNSUPPORTED;
  if (M > 0 && (!grad_y || !x || !mean || !rstd)) return GSAGE_ERR_INVALID_ARG;
  if (grad_weight || grad_bias) {
    if (!ws) return GSAGE_ERR_INVALID_ARG;
    if (ws_bytes < gsage_layer_norm_bwd_workspace_bytes(M, F, dtype)) return GSAGE_ERR_WORKSPACE;
  }
  const Drop d{p, 1.0f / (1.0f - p), seed, seed_dev};
  const auto go = dtype == GSAGE_F32 ? ln_bwd<float> : dtype == GSAGE_BF16 ? ln_bwd<__bf16> : ln_bwd<_Float16>;
  return go(grad_y, grad_sum, x, residual, weight, mean, rstd, M, F, wdtype, d, grad_x, grad_residual, grad_weight,
            grad_bias, (float *)ws, gs_stream(stream));
}
