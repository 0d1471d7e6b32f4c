// Shared helpers of the operators of the networks that the loss trains
// (recurrence, residual norms, optimizer): element types, conversions, sums.
#pragma once

#include "common.hpp"

namespace pesq {

using bf16 = __bf16;
using f16 = _Float16;

__host__ inline bool known_type(int dtype) {
    return dtype == PESQ_F32 || dtype == PESQ_BF16 || dtype == PESQ_F16;
}
__host__ inline int type_size(int dtype) { return dtype == PESQ_F32 ? 4 : 2; }

// fn(T()) with the element type of a PESQ_F32 / PESQ_BF16 / PESQ_F16 code
template <class Fn>
void with_type(int dtype, Fn fn) {
    if (dtype == PESQ_F32) {
        fn(float());
    } else if (dtype == PESQ_BF16) {
        fn(bf16());
    } else {
        fn(f16());
    }
}

// 2^x and log2(x) by the hardware's instructions (one unit in the last place,
// results below the normal range are flushed), and 1/x likewise
__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }
__device__ __forceinline__ float log2_fast(float x) { return __builtin_amdgcn_logf(x); }
__device__ __forceinline__ float rcp_fast(float x) { return __builtin_amdgcn_rcpf(x); }

constexpr float kLog2e = 1.44269504088896340736f;
constexpr float kLn2 = 0.69314718055994530942f;

__device__ __forceinline__ float sigmoid_fast(float x) {
    return rcp_fast(1.0f + exp2_fast(-kLog2e * x));
}

}  // namespace pesq
