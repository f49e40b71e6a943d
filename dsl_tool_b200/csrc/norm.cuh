// Host launchers of the row-wise kernels in norm.cu.
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

namespace dsl {
cudaError_t launch_quant_int8(const void* x, int dtype, long long rows, int cols, float* scale_out, int8_t* q, cudaStream_t st);
cudaError_t launch_rms_norm(const void* x, int dtype, long long rows, int cols, const void* residual, const void* gain, int gain_dtype,
                            float eps, int out_format, void* sum_out, void* out, float* scale_out, const float* scale_in,
                            cudaStream_t st);
}  // namespace dsl
