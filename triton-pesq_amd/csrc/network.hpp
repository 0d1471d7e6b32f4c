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

// 2^x by the hardware's instruction (one unit in the last place,
// results below the normal range are flushed), and 1/x likewise
__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }
__device__ __forceinline__ float rcp_fast(float x) { return __builtin_amdgcn_rcpf(x); }

constexpr float kLog2e = 1.44269504088896340736f;
constexpr float kLn2 = 0.69314718055994530942f;

// The exponent is rounded once: the relative error grows with |x| for negative x
// (3e-7 at -5, 1e-6 at -20, where the sigmoid is 2e-9), the absolute one does not.
__device__ __forceinline__ float sigmoid_fast(float x) {
    return rcp_fast(1.0f + exp2_fast(-kLog2e * x));
}

// V neighbouring elements moved at once from and to any element of a tensor:
// the hardware takes 16 byte accesses at any address, so rows of odd lengths
// need no element by element variant, only their ends do.
template <class T, int V>
struct Neighbours {
    T v[V];
};

template <class T, int V>
__device__ __forceinline__ Neighbours<T, V> load_neighbours(const T *p) {
    constexpr int kBytes = sizeof(T) * V, kMove = kBytes < 16 ? kBytes : 16;
    typedef uint32_t __attribute__((ext_vector_type(kMove / 4), aligned(sizeof(T)))) Move;
    struct Moves {
        Move m[kBytes / kMove];
    } moves;
#pragma unroll
    for (int k = 0; k < kBytes / kMove; ++k) moves.m[k] = reinterpret_cast<const Move *>(p)[k];
    return __builtin_bit_cast(Neighbours<T, V>, moves);
}

template <class T, int V>
__device__ __forceinline__ void store_neighbours(T *p, const Neighbours<T, V> &e) {
    constexpr int kBytes = sizeof(T) * V, kMove = kBytes < 16 ? kBytes : 16;
    typedef uint32_t __attribute__((ext_vector_type(kMove / 4), aligned(sizeof(T)))) Move;
    struct Moves {
        Move m[kBytes / kMove];
    };
    const Moves moves = __builtin_bit_cast(Moves, e);
#pragma unroll
    for (int k = 0; k < kBytes / kMove; ++k) reinterpret_cast<Move *>(p)[k] = moves.m[k];
}

// Sums of columns of partial sums [parts][stride] by a workgroup of kSumShares
// threads for each of kSumColumns columns: shares of the parts first, then their
// sums pairwise in LDS.  Returns column `c`'s (c < columns) to the threads of
// share 0.  Many shares, since the time is that of a thread's loads in a row.
constexpr int kSumShares = 64, kSumColumns = 16;

__device__ __forceinline__ float sum_parts(const float *part, int64_t parts, int64_t stride, int64_t c,
                                           int64_t columns) {
    __shared__ float sums[kSumShares][kSumColumns];
    const int column = threadIdx.x % kSumColumns, share = threadIdx.x / kSumColumns;
    float sum = 0.0f;
    if (c < columns) {
#pragma unroll 8
        for (int64_t k = share; k < parts; k += kSumShares) sum += part[k * stride + c];
    }
    sums[share][column] = sum;
    for (int half = kSumShares / 2; half > 0; half /= 2) {
        __syncthreads();
        if (share < half) sums[share][column] += sums[share + half][column];
    }
    return sums[0][column];
}

}  // namespace pesq
