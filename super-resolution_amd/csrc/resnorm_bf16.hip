// The residual-branch norms for bfloat16 tensors (resnorm_kernels.h; a file of its own to build beside the other type's).
#include "resnorm_kernels.h"

int resnorm::launch_bf16(const Plan& p, int backward, hipStream_t s) { return launch<bf16>(p, backward, s); }
