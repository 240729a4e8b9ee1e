// Host entry points of the norm kernels (norm.cu); the C ABI in api.cu wraps them.
#pragma once
#include <cuda_runtime.h>
#include <stddef.h>

#include "../../include/gpa_b200.h"

namespace gpa {

int norm_forward(const GpaNormArgs* a, void* stream_out, void* normed, cudaStream_t st, const char** why);
size_t norm_scratch_bytes(const GpaNormArgs* a);
int norm_backward(const GpaNormArgs* a, const void* stream_in, const void* dstream, const void* dnormed,
                  const GpaNormGrads* g, void* scratch, size_t scratch_bytes, cudaStream_t st,
                  const char** why);

}  // namespace gpa
