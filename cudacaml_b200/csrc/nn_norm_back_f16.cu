// The gradient's kernels for f16.
#include "nn_norm_back.cuh"

namespace ccb_nn {
void backward_f16(int x_dtype, int kind, const BackP& p, int sms, cudaStream_t st) { by_f16<Backward>(CCB_F16, x_dtype, kind, p, sms, st); }
}  // namespace ccb_nn
