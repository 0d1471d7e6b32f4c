// The end of a residual block and the start of the next, row by row:
//
//   y = branch silu(gate)        z = y / rms(y) post        (rms(v)^2 = mean v^2 + eps)
//   x' = x + scale z             n = x' / rms(x') next
//
// with any of gate, scale and next missing, or only the last (branch missing:
// n = x / rms(x) next).  Backward, with dx' and dn upstream and hats for the
// normalised rows:
//
//   v = dn next                  gx = dx' + (v - x'^ mean(v x'^)) / rms(x')
//   v = gx scale post            gy = (v - y^ mean(v y^)) / rms(y)
//   dx = gx     dbranch = gy silu(gate)     dgate = gy branch silu'(gate)
//   dpost = sum gx scale y^      dscale = sum gx post y^      dnext = sum dn x'^
//
// The backward reads x, branch and gate again instead of x' and n, so that x'
// need not be rounded; 1 / rms of both is kept from the forward.
#include <cmath>

#include "network.hpp"

namespace pesq {

constexpr int kNormThreads = 256;

struct NormArgs {
    int64_t rows, channels;
    const void *x, *branch, *gate;
    int64_t sx, sb, sg;
    const float *post, *scale, *next;
    float eps;
};

__device__ __forceinline__ float wave_sum32(float v) {
#pragma unroll
    for (int m = 32; m >= 1; m >>= 1) v += shfl_xor(v, m);
    return v;
}

// sum over the workgroup, to every thread; `scratch`: one float per wavefront
__device__ __forceinline__ float block_sum32(float v, float *scratch) {
    v = wave_sum32(v);
    __syncthreads();
    if (threadIdx.x % kWave == 0) scratch[threadIdx.x / kWave] = v;
    __syncthreads();
    float total = 0.0f;
    for (int w = 0; w < kNormThreads / kWave; ++w) total += scratch[w];
    return total;
}

template <class S, class T>
__global__ void __launch_bounds__(kNormThreads)
    residual_norm_fwd_kernel(NormArgs p, S *x_out, T *n_out, float *inv) {
    __shared__ float scratch[kNormThreads / kWave];
    const int64_t row = blockIdx.x;
    const S *x = static_cast<const S *>(p.x) + row * p.sx;
    const T *branch = static_cast<const T *>(p.branch) + row * p.sb;
    const T *gate = static_cast<const T *>(p.gate) + row * p.sg;
    const float count = static_cast<float>(p.channels);
    auto y_of = [&](int64_t c) {
        const float b = static_cast<float>(branch[c]);
        if (!p.gate) return b;
        const float g = static_cast<float>(gate[c]);
        return b * (g * sigmoid_fast(g));
    };
    float inv_y = 0.0f;
    if (p.branch) {
        float sum = 0.0f;
        for (int64_t c = threadIdx.x; c < p.channels; c += kNormThreads) {
            const float y = y_of(c);
            sum = fmaf(y, y, sum);
        }
        inv_y = 1.0f / sqrtf(block_sum32(sum, scratch) / count + p.eps);
        if (inv && threadIdx.x == 0) inv[2 * row] = inv_y;
    }
    auto x_of = [&](int64_t c) {
        const float v = static_cast<float>(x[c]);
        if (!p.branch) return v;
        const float z = y_of(c) * inv_y * p.post[c];
        return p.scale ? fmaf(p.scale[c], z, v) : v + z;
    };
    float sum = 0.0f;
    for (int64_t c = threadIdx.x; c < p.channels; c += kNormThreads) {
        const float v = x_of(c);
        if (x_out) x_out[row * p.channels + c] = static_cast<S>(v);
        sum = fmaf(v, v, sum);
    }
    if (!p.next) return;
    const float inv_x = 1.0f / sqrtf(block_sum32(sum, scratch) / count + p.eps);
    if (inv && threadIdx.x == 0) inv[2 * row + 1] = inv_x;
    for (int64_t c = threadIdx.x; c < p.channels; c += kNormThreads) {
        n_out[row * p.channels + c] = static_cast<T>(x_of(c) * inv_x * p.next[c]);
    }
}

// one workgroup per row; the row's shares of the weights' gradients go to
// part[row][3][channels]
template <class S, class T>
__global__ void __launch_bounds__(kNormThreads)
    residual_norm_bwd_kernel(NormArgs p, const S *g_out, int64_t sgo, const T *g_next, int64_t sgn,
                             const float *inv, S *g_x, T *g_branch, T *g_gate, float *part) {
    __shared__ float scratch[kNormThreads / kWave];
    const int64_t row = blockIdx.x;
    const S *x = static_cast<const S *>(p.x) + row * p.sx;
    const T *branch = static_cast<const T *>(p.branch) + row * p.sb;
    const T *gate = static_cast<const T *>(p.gate) + row * p.sg;
    const float count = static_cast<float>(p.channels);
    const float inv_y = inv[2 * row], inv_x = inv[2 * row + 1];
    auto y_of = [&](int64_t c) {
        const float b = static_cast<float>(branch[c]);
        if (!p.gate) return b;
        const float g = static_cast<float>(gate[c]);
        return b * (g * sigmoid_fast(g));
    };
    auto x_of = [&](int64_t c) {
        const float v = static_cast<float>(x[c]);
        if (!p.branch) return v;
        const float z = y_of(c) * inv_y * p.post[c];
        return p.scale ? fmaf(p.scale[c], z, v) : v + z;
    };
    const bool next = g_next != nullptr;
    float mean_x = 0.0f;
    if (next) {
        float sum = 0.0f;
        for (int64_t c = threadIdx.x; c < p.channels; c += kNormThreads) {
            sum = fmaf(static_cast<float>(g_next[row * sgn + c]) * p.next[c], x_of(c) * inv_x, sum);
        }
        mean_x = block_sum32(sum, scratch) / count;
    }
    auto gx_of = [&](int64_t c) {
        float g = g_out ? static_cast<float>(g_out[row * sgo + c]) : 0.0f;
        if (next) {
            const float v = static_cast<float>(g_next[row * sgn + c]) * p.next[c];
            g += inv_x * (v - x_of(c) * inv_x * mean_x);
        }
        return g;
    };
    float mean_y = 0.0f;
    if (p.branch) {
        float sum = 0.0f;
        for (int64_t c = threadIdx.x; c < p.channels; c += kNormThreads) {
            const float v = gx_of(c) * p.post[c] * (p.scale ? p.scale[c] : 1.0f);
            sum = fmaf(v, y_of(c) * inv_y, sum);
        }
        mean_y = block_sum32(sum, scratch) / count;
    }
    for (int64_t c = threadIdx.x; c < p.channels; c += kNormThreads) {
        const float g = gx_of(c);
        float *sums = part + (row * 3) * p.channels + c;
        if (next) sums[2 * p.channels] = static_cast<float>(g_next[row * sgn + c]) * x_of(c) * inv_x;
        if (g_x) g_x[row * p.channels + c] = static_cast<S>(g);
        if (!p.branch) continue;
        const float unit = y_of(c) * inv_y, scale = p.scale ? p.scale[c] : 1.0f;
        sums[0] = g * scale * unit;
        sums[p.channels] = g * p.post[c] * unit;
        const float gy = inv_y * (g * scale * p.post[c] - unit * mean_y);
        if (!p.gate) {
            if (g_branch) g_branch[row * p.channels + c] = static_cast<T>(gy);
            continue;
        }
        const float a = static_cast<float>(gate[c]), sig = sigmoid_fast(a);
        if (g_branch) g_branch[row * p.channels + c] = static_cast<T>(gy * a * sig);
        if (g_gate) {
            g_gate[row * p.channels + c] =
                static_cast<T>(gy * static_cast<float>(branch[c]) * sig * fmaf(a, 1.0f - sig, 1.0f));
        }
    }
}

// the three weights' gradients (blockIdx.y; NULL: none) from their partial sums
__global__ void __launch_bounds__(kNormThreads)
    residual_norm_sum_kernel(const float *part, int64_t parts, int64_t channels, float *g_post,
                             float *g_scale, float *g_next) {
    const int64_t c = int64_t(blockIdx.x) * kNormThreads + threadIdx.x;
    float *out = blockIdx.y == 0 ? g_post : blockIdx.y == 1 ? g_scale : g_next;
    if (c >= channels || !out) return;
    double sum = 0.0;
    for (int64_t k = 0; k < parts; ++k) sum += part[(3 * k + blockIdx.y) * channels + c];
    out[c] = static_cast<float>(sum);
}

// ---------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------

constexpr int64_t kMaxChannels = 8192;

static int check_norm(const pesq_residual_norm *p) {
    PESQ_CHECK_ARG(p != nullptr, "null argument");
    PESQ_CHECK_ARG(known_type(p->dtype) && known_type(p->stream_dtype), "unknown element type");
    PESQ_CHECK_ARG(p->stream_dtype == p->dtype || p->stream_dtype == PESQ_F32,
                   "the stream's type has to be float32 or the branch's");
    PESQ_CHECK_ARG(p->rows >= 0 && p->rows < (int64_t(1) << 31), "0 to 2^31 - 1 rows, got %lld",
                   (long long)p->rows);
    PESQ_CHECK_ARG(p->channels >= 1 && p->channels <= kMaxChannels,
                   "a residual norm has 1 to %lld channels, got %lld", (long long)kMaxChannels,
                   (long long)p->channels);
    PESQ_CHECK_ARG(p->eps >= 0.0 && std::isfinite(p->eps), "eps has to be finite and not negative");
    PESQ_CHECK_ARG(p->strides[0] >= 0 && p->strides[1] >= 0 && p->strides[2] >= 0, "negative stride");
    return PESQ_OK;
}

static int check_norm_operands(const pesq_residual_norm *p) {
    if (int st = check_norm(p)) return st;
    if (p->rows == 0) return PESQ_OK;  // tensors without elements have no address
    PESQ_CHECK_ARG(p->branch ? p->post_weight != nullptr : !p->gate && !p->scale && p->next_weight,
                   "a branch needs its weight; without one there is only the next weight");
    PESQ_CHECK_ARG(p->x, "null argument");
    return PESQ_OK;
}

static NormArgs norm_args(const pesq_residual_norm *p) {
    return {p->rows, p->channels, p->x, p->branch, p->gate, p->strides[0], p->strides[1],
            p->strides[2], p->post_weight, p->scale, p->next_weight, static_cast<float>(p->eps)};
}

// fn(S(), T()) with the stream's and the branch's types
template <class Fn>
static void with_types(const pesq_residual_norm *p, Fn fn) {
    with_type(p->dtype, [&](auto t) {
        if (p->stream_dtype == PESQ_F32) {
            fn(float(), t);
        } else {
            fn(t, t);
        }
    });
}

}  // namespace pesq

using namespace pesq;

extern "C" int pesq_residual_norm_workspace(const pesq_residual_norm *p, size_t *backward) {
    if (int st = check_norm(p)) return st;
    PESQ_CHECK_ARG(backward != nullptr, "null argument");
    *backward = size_t(p->rows) * 3 * p->channels * sizeof(float);
    return PESQ_OK;
}

extern "C" int pesq_residual_norm_forward(const pesq_residual_norm *p, void *x_out, void *n_out,
                                          float *inverse, hipStream_t stream) {
    if (int st = check_norm_operands(p)) return st;
    if (p->rows == 0) return PESQ_OK;
    PESQ_CHECK_ARG((!p->branch || x_out) && (!p->next_weight || n_out), "null argument");
    with_types(p, [&](auto s, auto t) {
        using S = decltype(s);
        using T = decltype(t);
        residual_norm_fwd_kernel<S, T><<<static_cast<unsigned>(p->rows), kNormThreads, 0, stream>>>(
            norm_args(p), p->branch ? static_cast<S *>(x_out) : nullptr, static_cast<T *>(n_out),
            inverse);
    });
    PESQ_CHECK_LAUNCH("pesq_residual_norm_forward");
    return PESQ_OK;
}

extern "C" int pesq_residual_norm_backward(const pesq_residual_norm *p, const void *g_x_out,
                                           const void *g_n_out, const int64_t *g_strides,
                                           const float *inverse, void *g_x, void *g_branch,
                                           void *g_gate, float *g_post, float *g_scale,
                                           float *g_next, void *workspace, hipStream_t stream) {
    if (int st = check_norm_operands(p)) return st;
    PESQ_CHECK_ARG(g_strides && g_strides[0] >= 0 && g_strides[1] >= 0, "the upstream strides");
    PESQ_CHECK_ARG(p->rows == 0 || (inverse && workspace), "null argument");
    PESQ_CHECK_ARG(!g_n_out || p->next_weight, "a gradient of n without its weight");
    PESQ_CHECK_ARG(p->rows == 0 || ((p->branch || (!g_branch && !g_post)) && (p->gate || !g_gate) &&
                                     (p->scale || !g_scale) && (p->next_weight || !g_next)),
                   "a gradient is asked of an operand that is not there");
    float *part = static_cast<float *>(workspace);
    if (p->rows > 0) {
        with_types(p, [&](auto s, auto t) {
            using S = decltype(s);
            using T = decltype(t);
            residual_norm_bwd_kernel<S, T>
                <<<static_cast<unsigned>(p->rows), kNormThreads, 0, stream>>>(
                    norm_args(p), static_cast<const S *>(g_x_out), g_strides[0],
                    static_cast<const T *>(g_n_out), g_strides[1], inverse, static_cast<S *>(g_x),
                    static_cast<T *>(g_branch), static_cast<T *>(g_gate), part);
        });
        PESQ_CHECK_LAUNCH("pesq_residual_norm_backward");
    }
    if (g_post || g_scale || g_next) {
        PESQ_CHECK_ARG(!g_next || g_n_out || p->rows == 0, "the next weight's gradient without n's");
        residual_norm_sum_kernel<<<dim3(static_cast<unsigned>(cdiv(p->channels, kNormThreads)), 3),
                                   kNormThreads, 0, stream>>>(part, p->rows, p->channels, g_post,
                                                              g_scale, g_next);
        PESQ_CHECK_LAUNCH("pesq_residual_norm_backward");
    }
    return PESQ_OK;
}
