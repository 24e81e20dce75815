// Layer norm and dropout on bf16 tables.
#include "norm_kernels.h"

int norm_dropout_bf16(const void *x, int64_t n, const NormDrop &d, void *out, hipStream_t st) {
  return dropout_go<__bf16>(x, n, d, out, st);
}
int norm_fwd_bf16(const NormFwd &n, hipStream_t st) { return ln_fwd<__bf16>(n, st); }
int norm_bwd_bf16(const NormBwd &n, hipStream_t st) { return ln_bwd<__bf16>(n, st); }
