// The two forms of linear attention over a prompt: chunks on the tensor cores (linear_chunk.cu), and the recurrence
// token by token (linear_attention.cu).
#pragma once

#include "common.cuh"

namespace sc {
namespace lc {
bool takes(const sc_linear& a);
size_t workspace(const sc_linear& a);
int launch(const sc_linear& a, void* workspace, int* err, cudaStream_t stream);
}  // namespace lc
}  // namespace sc
