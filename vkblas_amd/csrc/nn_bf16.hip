// nn_bf16.hip — the gated projection and linear cross entropy inside the
// pipelined GEMM kernel, bf16 operands.
#include "nn_pipe.hpp"

VKB_NN_TYPE(bf16, __bf16)
