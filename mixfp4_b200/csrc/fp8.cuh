// Shared by the block-scaled E4M3 quantizer and product (fp8_quantize.cu, fp8_gemm.cu).
#pragma once

#include "common.cuh"

namespace mixfp4 {

constexpr int kFp8Block = 128;
// Rows that a scale array of activations has room for: the product fetches the scales of up to 128 rows at once.
__host__ __device__ inline int64_t fp8_scale_rows(int64_t m) { return (m + 127) / 128 * 128; }

// Arguments of mixfp4_fp8_quantize_rows, checked before any CUDA call; then the pass itself.
int fp8_check_rows(const void* x, int dtype, int64_t m, int64_t k, int64_t ldx, const uint8_t* codes, int64_t ldq,
                   const float* scales, int64_t lds);
int fp8_quantize_rows(const void* x, int dtype, int64_t m, int64_t k, int64_t ldx, uint8_t* codes, int64_t ldq,
                      float* scales, int64_t lds, cudaStream_t st);

}  // namespace mixfp4
