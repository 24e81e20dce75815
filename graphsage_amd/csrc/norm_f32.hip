// Layer norm and dropout on fp32 tables.
#include "norm_kernels.h"

int norm_dropout_f32(const void *x, int64_t n, const NormDrop &d, void *out, hipStream_t st) {
  return dropout_go<float>(x, n, d, out, st);
}
int norm_fwd_f32(const NormFwd &n, hipStream_t st) { return ln_fwd<float>(n, st); }
int norm_bwd_f32(const NormBwd &n, hipStream_t st) { return ln_bwd<float>(n, st); }
