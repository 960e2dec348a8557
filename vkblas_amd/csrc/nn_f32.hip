// nn_f32.hip — the gated projection and linear cross entropy inside the
// pipelined GEMM kernel, f32 operands.
#include "nn_pipe.hpp"

VKB_NN_TYPE(f32, float)
