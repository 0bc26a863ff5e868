// Tensor maps over what attention reads: rows of tokens with heads side by side, and pages.
#pragma once

#include <cstddef>

#include <cuda.h>
#include <cuda_fp16.h>
#include <cuda_runtime_api.h>

namespace fb {

// (column, head, row) of a matrix of token rows, boxes of `box_heads` heads of `box_rows` rows.
cudaError_t encode_rows(CUtensorMap* map, const __half* base, int heads, int rows, long long stride, int box_heads,
                        int box_rows);

// (column, row) of rows of 64 values without gaps.
cudaError_t encode_pages(CUtensorMap* map, const __half* base, long long rows, int box_rows);

}  // namespace fb
