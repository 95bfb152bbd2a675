// host_operators.h -- the operators for fields of several experts, as the C ABI calls them (host_operators.cpp)
#pragma once
#include "host.h"
#include "operators.h"

namespace sng_host {

uint64_t expert_sort_workspace(uint32_t n, uint32_t k, uint32_t n_experts);
void expert_sort(sng_ctx* c, const int32_t* experts, uint32_t n, uint32_t k, uint32_t n_experts, int32_t* offsets, int32_t* order, int32_t* slot, void* workspace,
                 uint64_t workspace_bytes, hipStream_t s);
void expert_dispatch(sng_ctx* c, const void* x, int32_t dtype, uint32_t d, uint64_t ld_x, const int32_t* order, const int32_t* slot, uint32_t n, uint32_t k, void* rows,
                     uint64_t ld_rows, hipStream_t s);
void expert_combine(sng_ctx* c, const void* rows, int32_t dtype, uint32_t d, uint64_t ld_rows, const float* weights, const int32_t* slot, uint32_t n, uint32_t k, void* y,
                    uint64_t ld_y, hipStream_t s);
void expert_combine_backward(sng_ctx* c, const void* dy, uint64_t ld_dy, const void* rows, uint64_t ld_rows, int32_t dtype, uint32_t d, const float* weights,
                             const int32_t* slot, uint32_t n, uint32_t k, void* drows, uint64_t ld_drows, float* dweights, hipStream_t s);
void quantize_rows_i8(sng_ctx* c, const void* x, int32_t dtype, uint32_t rows, uint32_t cols, uint64_t ld_x, int8_t* q, uint64_t ld_q, float* scale, hipStream_t s);
uint64_t linear_i8_workspace(uint32_t rows, uint32_t n_in, uint32_t n_out, int32_t x_dtype, uint32_t n_experts);
void linear_i8(sng_ctx* c, const sng_linear_i8_args* a, hipStream_t s);

}  // namespace sng_host
