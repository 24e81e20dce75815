// Layer norm and dropout on fp16 tables.
#include "norm_kernels.h"

int norm_dropout_f16(const void *x, int64_t n, const NormDrop &d, void *out, hipStream_t st) {
  return dropout_go<_Float16>(x, n, d, out, st);
}
int norm_fwd_f16(const NormFwd &n, hipStream_t st) { return ln_fwd<_Float16>(n, st); }
int norm_bwd_f16(const NormBwd &n, hipStream_t st) { return ln_bwd<_Float16>(n, st); }
