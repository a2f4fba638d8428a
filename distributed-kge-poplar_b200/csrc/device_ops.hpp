// Launches of the operators on device arrays (device_ops.cu), checked and wrapped by the C ABI.
#pragma once

#include <cuda_runtime.h>

#include "common.hpp"

namespace kge {

size_t log_probs_workspace(size_t rows, size_t cols, size_t n_best);
void log_probs(const kge_scores& scores, const kge_log_probs_out& out, void* workspace, size_t workspace_bytes, cudaStream_t stream);
void log_probs_grad(const kge_scores& scores, const float* row_state, const float* grad_log_prob, const float* grad_entropy, size_t n_best,
                    const int32_t* best_index, const float* grad_best, void* grad_x, long long grad_row_stride, cudaStream_t stream);

void rows8_bytes(size_t rows, size_t cols, size_t* values, size_t* exponents);
void quantise_rows(const void* x, int float_type, size_t rows, size_t cols, long long row_stride, bool transposed, uint8_t* values,
                   uint8_t* exponents, cudaStream_t stream);
size_t product8_workspace(size_t m, size_t n, size_t k);
void product8(const uint8_t* a_values, const uint8_t* a_exponents, size_t m, const uint8_t* b_values, const uint8_t* b_exponents, size_t n,
              size_t k, void* out, int out_type, long long out_row_stride, void* workspace, size_t workspace_bytes, cudaStream_t stream);
bool product8_gave_up();

void adamw_step(const kge_adamw_args& args, const kge_adamw_tensor* tensors, size_t n_tensors, cudaStream_t stream);
uint32_t adamw_key(uint32_t seed, uint32_t step);
void adamw_moments(const uint8_t* adam_m, const uint8_t* m_exponent, const uint8_t* adam_v, const uint8_t* v_exponent, size_t size, void* m_bf16,
                   void* v_bf16, cudaStream_t stream);

}  // namespace kge
