// Products with 4-bit weights: fp16 activations.
#include "gemm_w4_kernels.h"

int nkl::w4_launch_f16(const W4Args& p, const W4Plan& pl, hipStream_t st) { return w4_launch<f16>(p, pl, st); }
