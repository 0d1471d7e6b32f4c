// Gated linear recurrence over time, diagonal over channels, with its backward:
//
//   u_t = rate softplus(decay) sigmoid(r_t),  a_t = exp(-u_t),  s_t = sqrt(1 - a_t^2)
//   h_t = a_t h_{t-1} + s_t sigmoid(i_t) x_t        (a_t h_{t-1} dropped at a reset)
//
// and with G_t = dy_t + a_{t+1} G_{t+1} in the opposite direction
//
//   dx_t = G_t s_t sigmoid(i_t)      di_t = G_t s_t x_t sigmoid(i_t) (1 - sigmoid(i_t))
//   du_t = G_t (a_t^2 / s_t sigmoid(i_t) x_t - a_t h_{t-1})       (h dropped at a reset)
//   dr_t = du_t u_t (1 - sigmoid(r_t))
//   ddecay = rate sigmoid(decay) sum_t du_t sigmoid(r_t)          dh_0 = a_1 G_1
//
// One thread per channel of a batch item walks along time.  The forward keeps
// the state before every kSteps steps, from which the backward runs them
// again: the states themselves are neither stored nor rounded.
#include <cmath>

#include "network.hpp"

namespace pesq {

constexpr int kSteps = 16;        // steps between two kept states
constexpr int kRecThreads = 64;

struct RecArgs {
    int64_t batch, time, channels;
    const void *x, *r, *i;
    int64_t sxb, sxt, srb, srt, sib, sit;
    const float *decay, *initial;
    const uint8_t *reset;
    float rate;
    bool reverse;
};

struct Rate {
    float k;       // log2 of the decay at an open gate, <= 0
    float factor;  // d u / d decay at an open gate: rate sigmoid(decay)
};

// rate softplus(decay), the logarithm of 1 + y as y log(w) / (w - 1), w = 1 + y
// rounded, which is exact where y is small
__device__ __forceinline__ Rate channel_rate(float decay, float rate) {
    const float y = exp2_fast(-kLog2e * fabsf(decay));
    const float w = 1.0f + y;
    const float log1p = w == 1.0f ? y : kLn2 * log2_fast(w) * y * rcp_fast(w - 1.0f);
    return {-(fmaxf(decay, 0.0f) + log1p) * rate * kLog2e, rate * sigmoid_fast(decay)};
}

// -expm1(-w) / w on [0, 0.5]: the polynomial of least largest relative error
constexpr float kP0 = 0.99999994039f, kP1 = -0.49999248981f, kP2 = 0.16654814780f,
                kP3 = -0.04100127891f, kP4 = 0.00677103782f;

struct Gates {
    float open_r, open_i, log2a, a, s;
};

// 1 - a^2 = -expm1(-w), w = 2 u: for small w by w (1 - w/2 + w^2/6 - ...), where
// the difference would cancel
__device__ __forceinline__ Gates gates(float r, float i, const Rate &c) {
    Gates g;
    g.open_r = sigmoid_fast(r);
    g.open_i = sigmoid_fast(i);
    g.log2a = c.k * g.open_r;
    g.a = exp2_fast(g.log2a);
    const float w = -2.0f * kLn2 * g.log2a;
    float p = kP4;
    p = fmaf(p, w, kP3);
    p = fmaf(p, w, kP2);
    p = fmaf(p, w, kP1);
    p = fmaf(p, w, kP0);
    const float square = w < 0.5f ? p * w : fmaf(-g.a, g.a, 1.0f);
    g.s = __builtin_amdgcn_sqrtf(square);
    return g;
}

// element (b, t, c) of a tensor with the given strides
template <class T>
__device__ __forceinline__ const T *at(const void *p, int64_t b, int64_t sb, int64_t t, int64_t st,
                                       int64_t c) {
    return static_cast<const T *>(p) + b * sb + t * st + c;
}

template <class T>
__global__ void __launch_bounds__(kRecThreads)
    recurrence_fwd_kernel(RecArgs p, T *y, float *last, float *starts) {
    const int64_t c = int64_t(blockIdx.x) * kRecThreads + threadIdx.x, b = blockIdx.y;
    if (c >= p.channels) return;
    const Rate rate = channel_rate(p.decay[c], p.rate);
    const int64_t parts = cdiv(p.time, kSteps);
    float h = p.initial ? p.initial[b * p.channels + c] : 0.0f;
    for (int64_t n = 0; n < p.time; ++n) {
        const int64_t t = p.reverse ? p.time - 1 - n : n;
        if (starts && n % kSteps == 0) starts[(b * parts + n / kSteps) * p.channels + c] = h;
        const float r = *at<T>(p.r, b, p.srb, t, p.srt, c);
        const float i = *at<T>(p.i, b, p.sib, t, p.sit, c);
        const float x = *at<T>(p.x, b, p.sxb, t, p.sxt, c);
        const Gates g = gates(r, i, rate);
        const float in = g.s * g.open_i * x;
        h = p.reset && p.reset[b * p.time + t] ? in : fmaf(g.a, h, in);
        y[(b * p.time + t) * p.channels + c] = static_cast<T>(h);
    }
    if (last) last[b * p.channels + c] = h;
}

// the sum of each channel's share of ddecay over time goes to decay_part[b, c]
template <class T>
__global__ void __launch_bounds__(kRecThreads)
    recurrence_bwd_kernel(RecArgs p, const T *gy, int64_t sgb, int64_t sgt, const float *g_last,
                          const float *starts, T *gx, T *gr, T *gi, float *decay_part,
                          float *g_initial) {
    const int64_t c = int64_t(blockIdx.x) * kRecThreads + threadIdx.x, b = blockIdx.y;
    if (c >= p.channels) return;
    const Rate rate = channel_rate(p.decay[c], p.rate);
    const int64_t parts = cdiv(p.time, kSteps);
    float carry = g_last ? g_last[b * p.channels + c] : 0.0f;
    float sum = 0.0f;
    for (int64_t part = parts - 1; part >= 0; --part) {
        const int64_t n0 = part * kSteps;
        const int steps = p.time - n0 < kSteps ? static_cast<int>(p.time - n0) : kSteps;
        float before[kSteps];
        float h = starts[(b * parts + part) * p.channels + c];
        for (int n = 0; n < steps; ++n) {
            const int64_t t = p.reverse ? p.time - 1 - n0 - n : n0 + n;
            if (p.reset && p.reset[b * p.time + t]) h = 0.0f;
            before[n] = h;
            const Gates g = gates(*at<T>(p.r, b, p.srb, t, p.srt, c),
                                  *at<T>(p.i, b, p.sib, t, p.sit, c), rate);
            const float x = *at<T>(p.x, b, p.sxb, t, p.sxt, c);
            h = fmaf(g.a, h, g.s * g.open_i * x);
        }
        for (int n = steps - 1; n >= 0; --n) {
            const int64_t t = p.reverse ? p.time - 1 - n0 - n : n0 + n;
            const Gates g = gates(*at<T>(p.r, b, p.srb, t, p.srt, c),
                                  *at<T>(p.i, b, p.sib, t, p.sit, c), rate);
            const float x = *at<T>(p.x, b, p.sxb, t, p.sxt, c);
            const float up = gy ? static_cast<float>(*at<T>(gy, b, sgb, t, sgt, c)) : 0.0f;
            const float grad = up + carry;
            const float driven = grad * g.open_i * x;
            // a^2 / s is infinite where u is 0; times u (1 - open) it tends to 0
            const float slope = g.s > 0.0f ? g.a * g.a * rcp_fast(g.s) : 0.0f;
            const float du = slope * driven - g.a * before[n] * grad;
            const int64_t out = (b * p.time + t) * p.channels + c;
            if (gx) gx[out] = static_cast<T>(grad * g.s * g.open_i);
            if (gi) gi[out] = static_cast<T>(driven * g.s * (1.0f - g.open_i));
            if (gr) gr[out] = static_cast<T>(du * (-kLn2 * g.log2a) * (1.0f - g.open_r));
            sum += du * g.open_r;
            carry = p.reset && p.reset[b * p.time + t] ? 0.0f : g.a * grad;
        }
    }
    decay_part[b * p.channels + c] = sum;
    if (g_initial) g_initial[b * p.channels + c] = carry;
}

__global__ void __launch_bounds__(kRecThreads)
    recurrence_decay_kernel(const float *part, int64_t rows, int64_t channels, const float *decay,
                            float rate, float *g_decay) {
    const int64_t c = int64_t(blockIdx.x) * kRecThreads + threadIdx.x;
    if (c >= channels) return;
    float sum = 0.0f;
    for (int64_t b = 0; b < rows; ++b) sum += part[b * channels + c];
    g_decay[c] = sum * channel_rate(decay[c], rate).factor;
}

template <class T>
__global__ void __launch_bounds__(kRecThreads) recurrence_step_kernel(RecArgs p, float *state, T *y) {
    const int64_t c = int64_t(blockIdx.x) * kRecThreads + threadIdx.x, b = blockIdx.y;
    if (c >= p.channels) return;
    const Gates g = gates(*at<T>(p.r, b, p.srb, 0, 0, c), *at<T>(p.i, b, p.sib, 0, 0, c),
                          channel_rate(p.decay[c], p.rate));
    const float x = *at<T>(p.x, b, p.sxb, 0, 0, c);
    const float h = fmaf(g.a, state[b * p.channels + c], g.s * g.open_i * x);
    state[b * p.channels + c] = h;
    y[b * p.channels + c] = static_cast<T>(h);
}

// ---------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------

static int check_recurrence(const pesq_recurrence *p) {
    PESQ_CHECK_ARG(p != nullptr, "null argument");
    PESQ_CHECK_ARG(known_type(p->dtype), "unknown element type %d", int(p->dtype));
    PESQ_CHECK_ARG(p->batch >= 0 && p->time >= 0 && p->channels >= 0,
                   "a recurrence has sizes of 0 or more, got %lld x %lld x %lld",
                   (long long)p->batch, (long long)p->time, (long long)p->channels);
    PESQ_CHECK_ARG(p->batch <= 65535, "a recurrence has at most 65535 batch items, got %lld",
                   (long long)p->batch);
    PESQ_CHECK_ARG(p->channels <= (int64_t(1) << 24) && p->time <= (int64_t(1) << 32),
                   "a recurrence has at most 2^24 channels and 2^32 steps, got %lld and %lld",
                   (long long)p->channels, (long long)p->time);
    PESQ_CHECK_ARG(p->rate > 0.0 && std::isfinite(p->rate), "the rate has to be positive and finite");
    for (int k = 0; k < 6; ++k) {
        PESQ_CHECK_ARG(p->strides[k / 2][k % 2] >= 0, "negative stride");
    }
    return PESQ_OK;
}

static bool empty(const pesq_recurrence *p) { return p->batch == 0 || p->channels == 0; }

static int check_operands(const pesq_recurrence *p) {
    if (int st = check_recurrence(p)) return st;
    if (empty(p)) return PESQ_OK;
    PESQ_CHECK_ARG(p->decay && (p->time == 0 || (p->x && p->recur_gate && p->input_gate)),
                   "null argument");
    return PESQ_OK;
}

static RecArgs kernel_args(const pesq_recurrence *p) {
    return {p->batch, p->time, p->channels, p->x, p->recur_gate, p->input_gate,
            p->strides[0][0], p->strides[0][1], p->strides[1][0], p->strides[1][1],
            p->strides[2][0], p->strides[2][1], p->decay, p->initial, p->reset,
            static_cast<float>(p->rate), p->reverse != 0};
}

static dim3 grid_of(const pesq_recurrence *p) {
    return dim3(static_cast<unsigned>(cdiv(p->channels, kRecThreads)),
                static_cast<unsigned>(p->batch));
}

}  // namespace pesq

using namespace pesq;

extern "C" int pesq_recurrence_workspace(const pesq_recurrence *p, size_t *starts, size_t *forward,
                                         size_t *backward) {
    if (int st = check_recurrence(p)) return st;
    const size_t states = size_t(p->batch) * p->channels * sizeof(float);
    if (starts) *starts = states * cdiv(p->time, kSteps);
    if (forward) *forward = 0;
    if (backward) *backward = states;
    return PESQ_OK;
}

extern "C" int pesq_recurrence_forward(const pesq_recurrence *p, void *y, float *last,
                                       float *starts, void *workspace, hipStream_t stream) {
    if (int st = check_operands(p)) return st;
    if (empty(p)) return PESQ_OK;
    PESQ_CHECK_ARG(y || p->time == 0, "null argument");
    with_type(p->dtype, [&](auto type) {
        using T = decltype(type);
        recurrence_fwd_kernel<T><<<grid_of(p), kRecThreads, 0, stream>>>(
            kernel_args(p), static_cast<T *>(y), last, starts);
    });
    PESQ_CHECK_LAUNCH("pesq_recurrence_forward");
    return PESQ_OK;
}

extern "C" int pesq_recurrence_backward(const pesq_recurrence *p, const void *g_y,
                                        const int64_t *g_strides, const float *g_last,
                                        const float *starts, void *g_x, void *g_recur,
                                        void *g_input, float *g_decay, float *g_initial,
                                        void *workspace, hipStream_t stream) {
    if (int st = check_operands(p)) return st;
    PESQ_CHECK_ARG(!g_y || (g_strides && g_strides[0] >= 0 && g_strides[1] >= 0),
                   "the upstream gradient needs its strides");
    if (p->channels == 0) return PESQ_OK;
    PESQ_CHECK_ARG(empty(p) || (workspace && (starts || p->time == 0)), "null argument");
    float *part = static_cast<float *>(workspace);
    if (p->batch > 0) {
        with_type(p->dtype, [&](auto type) {
            using T = decltype(type);
            recurrence_bwd_kernel<T><<<grid_of(p), kRecThreads, 0, stream>>>(
                kernel_args(p), static_cast<const T *>(g_y), g_y ? g_strides[0] : 0,
                g_y ? g_strides[1] : 0, g_last, starts, static_cast<T *>(g_x),
                static_cast<T *>(g_recur), static_cast<T *>(g_input), part, g_initial);
        });
        PESQ_CHECK_LAUNCH("pesq_recurrence_backward");
    }
    if (g_decay) {
        PESQ_CHECK_ARG(p->decay, "null argument");
        recurrence_decay_kernel<<<static_cast<unsigned>(cdiv(p->channels, kRecThreads)), kRecThreads,
                                  0, stream>>>(part, p->batch, p->channels, p->decay,
                                               static_cast<float>(p->rate), g_decay);
        PESQ_CHECK_LAUNCH("pesq_recurrence_backward");
    }
    return PESQ_OK;
}

extern "C" int pesq_recurrence_step(const pesq_recurrence *p, float *state, void *y,
                                    hipStream_t stream) {
    if (int st = check_operands(p)) return st;
    PESQ_CHECK_ARG(p->time == 1 && !p->reset, "a step is one frame without resets");
    if (empty(p)) return PESQ_OK;
    PESQ_CHECK_ARG(state && y, "null argument");
    with_type(p->dtype, [&](auto type) {
        using T = decltype(type);
        recurrence_step_kernel<T>
            <<<grid_of(p), kRecThreads, 0, stream>>>(kernel_args(p), state, static_cast<T *>(y));
    });
    PESQ_CHECK_LAUNCH("pesq_recurrence_step");
    return PESQ_OK;
}
