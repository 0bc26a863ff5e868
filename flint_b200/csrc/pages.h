// Error words of the kernels that keep a paged cache's tables and that select beams: numbers in device memory that were out
// of range.
#pragma once

#include <cuda_runtime_api.h>

namespace fb {

cudaError_t pages_error_flag(int* value, bool reset);
cudaError_t beams_error_flag(int* value, bool reset);

}  // namespace fb
