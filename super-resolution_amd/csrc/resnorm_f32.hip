// The residual-branch norms for float32 tensors (resnorm_kernels.h; a file of its own to build beside the other type's).
#include "resnorm_kernels.h"

int resnorm::launch_f32(const Plan& p, int backward, hipStream_t s) { return launch<float>(p, backward, s); }
