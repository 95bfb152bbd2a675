// operators.h -- device-side arguments and launchers of the operators for fields of several experts: samples sorted by
// expert and back (experts.hip), the 8-bit linear layer (linear_i8.hip).  host_operators.cpp checks the arguments.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "linear_i8_rule.h"

namespace sng {

enum { DT_F16 = 0, DT_BF16 = 1, DT_F32 = 2, DT_I8 = 3 };   // SNG_F16 ...

// n / d for n < 2^31 by one multiplication (Granlund & Montgomery, "Division by invariant integers using multiplication")
struct FastDiv {
    uint32_t mul = 0, shift = 0, d = 1;
    FastDiv() = default;
    explicit FastDiv(uint32_t div) : d(div) {
        while ((1ull << shift) < d) ++shift;
        mul = (uint32_t)(((1ull << 32) * ((1ull << shift) - d)) / d + 1);
    }
#ifdef __HIP_DEVICE_COMPILE__
    __device__ __forceinline__ uint32_t div(uint32_t n) const { return (__umulhi(n, mul) + n) >> shift; }
#else
    uint32_t div(uint32_t n) const { return (uint32_t)(((((uint64_t)n * mul) >> 32) + n) >> shift); }
#endif
};

// ---- samples by expert (experts.hip) ----------------------------------------------------------------------------
constexpr uint32_t EXPERTS_MAX = 4096;            // a wave's counters of every expert fit 16 KiB of LDS
constexpr uint32_t SORT_CHUNK = 4096;             // choices per workgroup of the sort that is not
constexpr uint32_t SORT_ONE_MAX = 16384;          // most choices that one workgroup sorts in one launch ...
constexpr uint32_t SORT_ONE_EXPERTS = 1024;       // ... over at most this many experts (16 waves x 4 KiB of LDS)
constexpr uint64_t CHOICES_MAX = 1ull << 28;

struct SortArgs {
    const int32_t* experts;
    uint32_t total, n_experts;   // total = n * k
    int32_t* offsets;
    int32_t* order;
    int32_t* slot;
    uint32_t* counts;            // workspace [blocks][n_experts], then [n_experts] totals
};
inline uint32_t sort_blocks(uint64_t total) { return total ? (uint32_t)((total + SORT_CHUNK - 1) / SORT_CHUNK) : 1u; }
inline bool sort_in_one(uint64_t total, uint32_t n_experts) { return total <= SORT_ONE_MAX && n_experts <= SORT_ONE_EXPERTS; }
void launch_expert_sort(const SortArgs& a, hipStream_t s);

struct RowsArgs {
    const void* src;         // x (dispatch), rows (combine, combine backward)
    uint64_t ld_src;         // elements
    void* dst;               // rows (dispatch), y (combine), drows (backward, may be null)
    uint64_t ld_dst;
    const void* dy;          // backward
    uint64_t ld_dy;
    const float* weights;    // null: ones
    float* dweights;         // backward, may be null
    const int32_t* slot;
    uint32_t n, k, d;
    int dtype;
};
void launch_expert_dispatch(const RowsArgs& a, hipStream_t s);
void launch_expert_combine(const RowsArgs& a, hipStream_t s);
void launch_expert_combine_backward(const RowsArgs& a, hipStream_t s);

// ---- 8-bit linear layer (linear_i8.hip) ---------------------------------------------------------------------------
constexpr uint32_t I8_IN_MAX = 131071;    // n_in * 128 * 128 < 2^31: the int32 sums cannot overflow
constexpr uint32_t I8_PAD = 128;          // bytes of a row that the tiles take at a time; the workspace's rows are padded to it

struct QuantArgs {
    const void* x;
    uint64_t ld_x;           // elements
    int dtype;
    uint32_t rows, cols, cols_written;   // q[cols .. cols_written) = 0
    int8_t* q;
    uint64_t ld_q;
    float* scale;            // not written for DT_I8
};
struct LinearArgs {
    const void* x;           // [rows][ld_x] of x_dtype
    uint64_t ld_x;           // elements
    int x_dtype;
    const float* x_scale;    // [rows], DT_I8
    const int8_t* w;         // [n_experts][n_out][ld_w]
    uint64_t ld_w;
    const float* w_scale;    // [n_experts][n_out]
    const float* bias;       // [n_experts][n_out] or null
    const int32_t* offsets;  // [n_experts + 1] rows of each expert, null: every row, one matrix
    uint32_t n_experts, rows, n_in, n_out;
    void* y;
    uint64_t ld_y;
    int y_dtype, relu;
    LinearKernel kernel;     // linear_i8_kernel's answer
    uint32_t splits;         // above 1: linear_i8_split's answer, and its workspace
    int32_t* partial;
};
// whether the kernel brings x to 8 bits itself (else x has to be DT_I8)
bool linear_i8_quantizes(uint32_t rows, uint32_t n_in, uint32_t n_out, uint32_t n_experts);
void launch_quantize_rows(const QuantArgs& a, hipStream_t s);
// rows of n >= 16 bytes at any place to rows of `padded` (a multiple of 16), zeros behind n
void launch_pad_rows(const int8_t* w, uint64_t ld_w, uint32_t n, uint64_t rows, uint32_t padded, int8_t* to, hipStream_t s);
void launch_linear_i8(const LinearArgs& a, hipStream_t s);

}  // namespace sng
