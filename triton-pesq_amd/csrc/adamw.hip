// One AdamW step over many tensors, moments in 32 or in 8 bits.
//
//   m = b1 m + (1 - b1) g          v = b2 v + (1 - b2) g^2
//   p = (1 - lr wd) p - lr / (1 - b1^t) m / (sqrt(v / (1 - b2^t)) + eps)
//
// in float32, each product and sum rounded as written (no fused steps), so that
// the result is the same however the elements are spread over threads.
//
// 8 bit moments are held in blocks of 256 elements of one tensor, each with its
// largest magnitude as a float32 scale, and per element the nearest
//
//   first moment    q = sign(m) round(127 sqrt(|m| / scale)),   m = scale q |q| / 127^2
//   second moment   q = round(255 (v / scale)^(1/4)),           v = scale q^4 / 255^4
//
// The roots spend the codes evenly over ratios rather than differences: a step
// is 1.6 % of a value near the scale in both, and the second moment, which
// spans squares, still has a step of 20 % at 4e-5 of the scale.  A second
// moment that is not 0 gets the code 1 at least, since 0 would put eps alone
// under the fraction.  The update itself uses the new moments before they are
// rounded.  Blocks whose scale is below 2^-100 are held as zeros: 1 / scale and
// the quotients would leave float32's range.  A NaN or infinite moment makes
// its block's scale NaN or infinite, so that it stays visible.
#include <cmath>

#include "network.hpp"

namespace pesq {

constexpr int kBlock = 256;  // elements per 8 bit scale
constexpr float kSmallest = 0x1p-100f;

struct AdamArgs {
    float b1, c1, b2, c2, keep, step_size, correction, eps;
};

// as written: no contraction into fused multiply-adds
#pragma clang fp contract(off)

struct Moments {
    float m, v;
};

__device__ __forceinline__ float adamw(float p, float g, Moments &s, const AdamArgs &a) {
    s.m = s.m * a.b1 + g * a.c1;
    s.v = s.v * a.b2 + (g * g) * a.c2;
    const float update = s.m / (sqrtf(s.v) * a.correction + a.eps);
    return p * a.keep - update * a.step_size;
}

__device__ __forceinline__ float value_m(int8_t q, float scale) {
    const float part = static_cast<float>(q) * (1.0f / 127.0f);
    return fabsf(part) * part * scale;
}

__device__ __forceinline__ float value_v(uint8_t q, float scale) {
    float part = static_cast<float>(q) * (1.0f / 255.0f);
    part = part * part;
    return part * part * scale;
}

__device__ __forceinline__ int8_t code_m(float m, float inverse) {
    const float q = rintf(sqrtf(fabsf(m) * inverse) * 127.0f);
    const int code = static_cast<int>(fminf(q, 127.0f));  // fmin: a NaN gives 127
    return static_cast<int8_t>(m < 0.0f ? -code : code);
}

__device__ __forceinline__ uint8_t code_v(float v, float inverse) {
    const float q = rintf(sqrtf(sqrtf(v * inverse)) * 255.0f);
    const int code = static_cast<int>(fminf(q, 255.0f));
    return static_cast<uint8_t>(v > 0.0f && inverse != 0.0f && code < 1 ? 1 : code);
}

// largest magnitude of the block, NaN above all (its bits are the largest)
__device__ __forceinline__ float block_scale(float v, uint32_t *scratch) {
    uint32_t bits = __float_as_uint(v) & 0x7fffffffu;
#pragma unroll
    for (int m = 32; m >= 1; m >>= 1) {
        const uint32_t other = __shfl_xor(bits, m, kWave);
        bits = other > bits ? other : bits;
    }
    __syncthreads();
    if (threadIdx.x % kWave == 0) scratch[threadIdx.x / kWave] = bits;
    __syncthreads();
    for (int w = 0; w < kBlock / kWave; ++w) bits = scratch[w] > bits ? scratch[w] : bits;
    const float scale = __uint_as_float(bits);
    return scale < kSmallest ? 0.0f : scale;
}

__device__ __forceinline__ float inverse_of(float scale) { return scale == 0.0f ? 0.0f : 1.0f / scale; }

template <class T>
__global__ void __launch_bounds__(kBlock)
    adamw32_kernel(T *p, const T *g, int64_t count, float *m, float *v, AdamArgs a) {
    const int64_t k = int64_t(blockIdx.x) * kBlock + threadIdx.x;
    if (k >= count) return;
    Moments s{m[k], v[k]};
    p[k] = static_cast<T>(adamw(static_cast<float>(p[k]), static_cast<float>(g[k]), s, a));
    m[k] = s.m;
    v[k] = s.v;
}

template <class T>
__global__ void __launch_bounds__(kBlock)
    adamw8_kernel(T *p, const T *g, int64_t count, int8_t *m, uint8_t *v, float *m_scale,
                  float *v_scale, AdamArgs a) {
    __shared__ uint32_t scratch[kBlock / kWave];
    const int64_t k = int64_t(blockIdx.x) * kBlock + threadIdx.x;
    Moments s{0.0f, 0.0f};
    if (k < count) {
        s = {value_m(m[k], m_scale[blockIdx.x]), value_v(v[k], v_scale[blockIdx.x])};
        p[k] = static_cast<T>(adamw(static_cast<float>(p[k]), static_cast<float>(g[k]), s, a));
    }
    const float sm = block_scale(s.m, scratch), sv = block_scale(s.v, scratch);
    if (threadIdx.x == 0) {
        m_scale[blockIdx.x] = sm;
        v_scale[blockIdx.x] = sv;
    }
    if (k >= count) return;
    m[k] = code_m(s.m, inverse_of(sm));
    v[k] = code_v(s.v, inverse_of(sv));
}

__global__ void __launch_bounds__(kBlock)
    adamw_moments_kernel(const int8_t *m, const uint8_t *v, const float *m_scale,
                         const float *v_scale, float *m_out, float *v_out) {
    const int64_t k = int64_t(blockIdx.x) * kBlock + threadIdx.x;
    m_out[k] = value_m(m[k], m_scale[blockIdx.x]);
    v_out[k] = value_v(v[k], v_scale[blockIdx.x]);
}

}  // namespace pesq

using namespace pesq;

extern "C" int pesq_adamw_step(const pesq_adamw_tensor *tensors, int64_t count,
                               const pesq_adamw_options *o, void *exp_avg, void *exp_avg_sq,
                               float *exp_avg_scale, float *exp_avg_sq_scale, hipStream_t stream) {
    PESQ_CHECK_ARG(o != nullptr && count >= 0 && (tensors || count == 0), "null argument");
    PESQ_CHECK_ARG(known_type(o->dtype), "unknown element type %d", int(o->dtype));
    PESQ_CHECK_ARG(o->state_bits == 32 || o->state_bits == 8, "moments have 32 or 8 bits, got %d",
                   int(o->state_bits));
    PESQ_CHECK_ARG(o->step >= 1, "steps count from 1, got %lld", (long long)o->step);
    PESQ_CHECK_ARG(o->beta1 >= 0.0 && o->beta1 < 1.0 && o->beta2 >= 0.0 && o->beta2 < 1.0,
                   "betas have to be in [0, 1)");
    const bool eight = o->state_bits == 8;
    PESQ_CHECK_ARG(count == 0 || (exp_avg && exp_avg_sq && (!eight || (exp_avg_scale && exp_avg_sq_scale))),
                   "null argument");
    for (int64_t k = 0; k < count; ++k) {
        PESQ_CHECK_ARG(tensors[k].count >= 0 && tensors[k].first >= 0 && tensors[k].first % kBlock == 0,
                       "tensor %lld has no place in the moments", (long long)k);
        PESQ_CHECK_ARG(tensors[k].count == 0 || (tensors[k].param && tensors[k].grad), "null argument");
        PESQ_CHECK_ARG(tensors[k].count < (int64_t(1) << 39), "tensor %lld is too large", (long long)k);
    }
    const double step = static_cast<double>(o->step);
    const AdamArgs a{static_cast<float>(o->beta1), static_cast<float>(1.0 - o->beta1),
                     static_cast<float>(o->beta2), static_cast<float>(1.0 - o->beta2),
                     static_cast<float>(1.0 - o->lr * o->weight_decay),
                     static_cast<float>(o->lr / (1.0 - std::pow(o->beta1, step))),
                     static_cast<float>(1.0 / std::sqrt(1.0 - std::pow(o->beta2, step))),
                     static_cast<float>(o->eps)};
    for (int64_t k = 0; k < count; ++k) {
        const pesq_adamw_tensor &t = tensors[k];
        if (t.count == 0) continue;
        const unsigned grid = static_cast<unsigned>(cdiv(t.count, kBlock));
        with_type(o->dtype, [&](auto type) {
            using T = decltype(type);
            if (eight) {
                adamw8_kernel<T><<<grid, kBlock, 0, stream>>>(
                    static_cast<T *>(t.param), static_cast<const T *>(t.grad), t.count,
                    static_cast<int8_t *>(exp_avg) + t.first,
                    static_cast<uint8_t *>(exp_avg_sq) + t.first, exp_avg_scale + t.first / kBlock,
                    exp_avg_sq_scale + t.first / kBlock, a);
            } else {
                adamw32_kernel<T><<<grid, kBlock, 0, stream>>>(
                    static_cast<T *>(t.param), static_cast<const T *>(t.grad), t.count,
                    static_cast<float *>(exp_avg) + t.first,
                    static_cast<float *>(exp_avg_sq) + t.first, a);
            }
        });
        PESQ_CHECK_LAUNCH("pesq_adamw_step");
    }
    return PESQ_OK;
}

extern "C" int pesq_adamw_moments(const void *exp_avg, const void *exp_avg_sq,
                                  const float *exp_avg_scale, const float *exp_avg_sq_scale,
                                  int64_t count, float *m, float *v, hipStream_t stream) {
    PESQ_CHECK_ARG(count >= 0 && count % kBlock == 0 && count < (int64_t(1) << 39),
                   "whole blocks of %d elements, got %lld", kBlock, (long long)count);
    if (count == 0) return PESQ_OK;
    PESQ_CHECK_ARG(exp_avg && exp_avg_sq && exp_avg_scale && exp_avg_sq_scale && m && v, "null argument");
    adamw_moments_kernel<<<static_cast<unsigned>(count / kBlock), kBlock, 0, stream>>>(
        static_cast<const int8_t *>(exp_avg), static_cast<const uint8_t *>(exp_avg_sq), exp_avg_scale,
        exp_avg_sq_scale, m, v);
    PESQ_CHECK_LAUNCH("pesq_adamw_moments");
    return PESQ_OK;
}
