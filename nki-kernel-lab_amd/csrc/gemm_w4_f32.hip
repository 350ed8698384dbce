// Products with 4-bit weights: fp32 activations.
#include "gemm_w4_kernels.h"

int nkl::w4_launch_f32(const W4Args& p, const W4Plan& pl, hipStream_t st) { return w4_launch<float>(p, pl, st); }
