// Products with 4-bit weights: bf16 activations.
#include "gemm_w4_kernels.h"

int nkl::w4_launch_bf16(const W4Args& p, const W4Plan& pl, hipStream_t st) { return w4_launch<bf16>(p, pl, st); }
