// nn_f16.hip — the gated projection and linear cross entropy inside the
// pipelined GEMM kernel, f16 operands.
#include "nn_pipe.hpp"

VKB_NN_TYPE(f16, _Float16)
