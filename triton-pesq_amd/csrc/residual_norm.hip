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
// need not be rounded; 1 / rms of both is kept from the forward.  dpost and
// dscale are one sum, sum gx y^, times the other weight.
//
// Memory bounds both passes (60016 x 1024, bfloat16 under a float32 stream: medians
// of 165 and 269 us, 5.2 and 5.0 TB/s).  A row is held in registers by 16 to 512 lanes, 8
// or 16 elements each, so that every tensor is read and written once; sums
// over a row go over lanes by DPP and, for rows of several wavefronts, over LDS.
// Workgroups walk over the rows with the weights in registers, and the
// backward's sums over rows stay in registers too, until one store per
// workgroup of partial sums, which a second kernel adds in a fixed order.
#include <cmath>
#include <type_traits>

#include "network.hpp"

namespace pesq {

constexpr int kNormThreads = 256;  // (512 for rows of more than 4096 channels)
constexpr int kMostNormThreads = 512;

struct NormArgs {
    int64_t rows, channels;
    const void *x, *branch, *gate;
    int64_t sx, sb, sg;
    const float *post, *scale, *next;
    float eps;
    int lanes;  // per row
    int whole;  // channels in whole vectors
};

template <int kCtrl>
__device__ __forceinline__ float dpp32(float v) {
    return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), kCtrl, 0xF, 0xF, true));
}

// sum over kWidth (16, 32 or 64) neighbouring lanes, to each of them, in a fixed order
template <int kWidth>
__device__ __forceinline__ float lanes_sum(float v) {
    v += dpp32<0x128>(v);  // row_ror:8, 4, 2, 1
    v += dpp32<0x124>(v);
    v += dpp32<0x122>(v);
    v += dpp32<0x121>(v);
    if constexpr (kWidth == 32) v += shfl_xor(v, 16);
    if constexpr (kWidth == 64) {
        const auto row = [&](int lane) {
            return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), lane));
        };
        v = (row(0) + row(16)) + (row(32) + row(48));
    }
    return v;
}

// Sums over the lanes of a row; over several wavefronts through two buffers in
// turn, so that one barrier a sum is enough.
template <int kWidth>
struct RowSum {
    float (*buffers)[kMostNormThreads / kWave];
    int waves, first;  // of the row
    int turn = 0;
    __device__ __forceinline__ float operator()(float v) {
        v = lanes_sum<kWidth>(v);
        if (kWidth < kWave || waves == 1) return v;
        float *buffer = buffers[turn];
        turn ^= 1;
        if (lane_id() == 0) buffer[wave_index()] = v;
        __syncthreads();
        v = 0.0f;
        for (int w = 0; w < waves; ++w) v += buffer[first + w];
        return v;
    }
};

// Where a thread stands: its lane of the row, and rows of the workgroup
struct NormPlace {
    int lane, group, groups;
    __device__ __forceinline__ explicit NormPlace(int lanes)
        : lane(threadIdx.x % lanes), group(threadIdx.x / lanes), groups(blockDim.x / lanes) {}
};

// N elements of a row by this thread: E in vectors of V neighbours, lanes V
// apart, and, where the row does not end with a vector (N = E + 1), one of the
// few left.  Zeros past the end.
template <int V, int E, int N, class T>
__device__ __forceinline__ void load_row(const T *row, const NormArgs &p, int lane, float (&out)[N]) {
#pragma unroll
    for (int j = 0; j < E / V; ++j) {
        const int c = (j * p.lanes + lane) * V;
        Neighbours<T, V> e{};
        if (c < p.whole) e = load_neighbours<T, V>(row + c);
#pragma unroll
        for (int k = 0; k < V; ++k) out[j * V + k] = static_cast<float>(e.v[k]);
    }
    if constexpr (N > E) {
        T t{};
        if (p.whole + lane < p.channels) t = row[p.whole + lane];
        out[E] = static_cast<float>(t);
    }
}

template <int V, int E, int N, class T>
__device__ __forceinline__ void store_row(T *row, const NormArgs &p, int lane, const float (&f)[N]) {
#pragma unroll
    for (int j = 0; j < E / V; ++j) {
        const int c = (j * p.lanes + lane) * V;
        Neighbours<T, V> e;
#pragma unroll
        for (int k = 0; k < V; ++k) e.v[k] = static_cast<T>(f[j * V + k]);
        if (c < p.whole) store_neighbours<T, V>(row + c, e);
    }
    if constexpr (N > E) {
        if (p.whole + lane < p.channels) row[p.whole + lane] = static_cast<T>(f[E]);
    }
}

// a weight by this thread, `otherwise` where there is none
template <int V, int E, int N>
__device__ __forceinline__ void load_weight(const float *w, const NormArgs &p, int lane, float otherwise,
                                            float (&out)[N]) {
    if (w) return load_row<V, E>(w, p, lane, out);
#pragma unroll
    for (int k = 0; k < N; ++k) out[k] = otherwise;
}

// use(channel, element) for each of a thread's elements, by vectors and alone
template <int V, int E, int N, class Use>
__device__ __forceinline__ void each_channel(const NormArgs &p, int lane, Use use) {
#pragma unroll
    for (int j = 0; j < E / V; ++j) {
        const int c = (j * p.lanes + lane) * V;
        if (c < p.whole) {
#pragma unroll
            for (int k = 0; k < V; ++k) use(c + k, j * V + k);
        }
    }
    if constexpr (N > E) {
        if (p.whole + lane < p.channels) use(p.whole + lane, E);
    }
}

// V: elements of a 16 byte move of T; E: of a thread in such; kTail: whether rows
// end with part of one
template <class S, class T, int V, int E, int kWidth, bool kTail>
__global__ void __launch_bounds__(kMostNormThreads)
    residual_norm_fwd_kernel(NormArgs p, S *x_out, T *n_out, float *inv) {
    __shared__ float buffers[2][kMostNormThreads / kWave];
    constexpr int N = E + kTail;
    const NormPlace at(p.lanes);
    RowSum<kWidth> row_sum{buffers, p.lanes / kWave, static_cast<int>(threadIdx.x) / p.lanes * (p.lanes / kWave)};
    const float share = 1.0f / static_cast<float>(p.channels);
    float both[N], next[N];
    if (p.branch) {
        load_weight<V, E>(p.post, p, at.lane, 1.0f, both);
        load_weight<V, E>(p.scale, p, at.lane, 1.0f, next);
#pragma unroll
        for (int k = 0; k < N; ++k) both[k] *= next[k];
    }
    load_weight<V, E>(p.next, p, at.lane, 1.0f, next);
    const int64_t step = int64_t(gridDim.x) * at.groups;
    for (int64_t first = int64_t(blockIdx.x) * at.groups; first < p.rows; first += step) {
        // (every lane takes part in the sums)
        const bool there = first + at.group < p.rows;
        const int64_t row = there ? first + at.group : p.rows - 1;
        float x[N], y[N];
        load_row<V, E>(static_cast<const S *>(p.x) + row * p.sx, p, at.lane, x);
        if (p.branch) {
            load_row<V, E>(static_cast<const T *>(p.branch) + row * p.sb, p, at.lane, y);
            if (p.gate) {
                float g[N];
                load_row<V, E>(static_cast<const T *>(p.gate) + row * p.sg, p, at.lane, g);
#pragma unroll
                for (int k = 0; k < N; ++k) y[k] *= g[k] * sigmoid_fast(g[k]);
            }
            float sum = 0.0f;
#pragma unroll
            for (int k = 0; k < N; ++k) sum = fmaf(y[k], y[k], sum);
            const float inv_y = 1.0f / sqrtf(fmaf(row_sum(sum), share, p.eps));
            if (inv && there && at.lane == 0) inv[2 * row] = inv_y;
#pragma unroll
            for (int k = 0; k < N; ++k) x[k] = fmaf(both[k], y[k] * inv_y, x[k]);
            if (there) store_row<V, E>(x_out + row * p.channels, p, at.lane, x);
        }
        if (p.next) {
            float sum = 0.0f;
#pragma unroll
            for (int k = 0; k < N; ++k) sum = fmaf(x[k], x[k], sum);
            const float inv_x = 1.0f / sqrtf(fmaf(row_sum(sum), share, p.eps));
            if (inv && there && at.lane == 0) inv[2 * row + 1] = inv_x;
#pragma unroll
            for (int k = 0; k < N; ++k) x[k] *= inv_x * next[k];
            if (there) store_row<V, E>(n_out + row * p.channels, p, at.lane, x);
        }
    }
}

// part[workgroup][2][channels]: the workgroup's sums of gx y^ and dn x'^
template <class S, class T, int V, int E, int kWidth, bool kTail>
__global__ void __launch_bounds__(kMostNormThreads)
    residual_norm_bwd_kernel(NormArgs p, const S *g_out, int64_t sgo, const T *g_next, int64_t sgn,
                             const float *inv, S *g_x, T *g_branch, T *g_gate, float *part) {
    __shared__ float buffers[2][kMostNormThreads / kWave];
    __shared__ float sums[2 * (E * kNormThreads / 2 + V)];  // (several groups: half the threads each at most)
    constexpr int N = E + kTail;
    const NormPlace at(p.lanes);
    RowSum<kWidth> row_sum{buffers, p.lanes / kWave, static_cast<int>(threadIdx.x) / p.lanes * (p.lanes / kWave)};
    const float share = 1.0f / static_cast<float>(p.channels);
    float both[N], next[N], sum_both[N], sum_next[N];
    load_weight<V, E>(p.post, p, at.lane, 1.0f, both);
    load_weight<V, E>(p.scale, p, at.lane, 1.0f, next);
#pragma unroll
    for (int k = 0; k < N; ++k) {
        both[k] *= next[k];
        sum_both[k] = sum_next[k] = 0.0f;
    }
    load_weight<V, E>(p.next, p, at.lane, 1.0f, next);
    const int64_t step = int64_t(gridDim.x) * at.groups;
    for (int64_t first = int64_t(blockIdx.x) * at.groups; first < p.rows; first += step) {
        const bool there = first + at.group < p.rows;
        const int64_t row = there ? first + at.group : p.rows - 1;
        float x[N], b[N], a[N], gx[N];
        load_row<V, E>(static_cast<const S *>(p.x) + row * p.sx, p, at.lane, x);
        if (p.branch) load_row<V, E>(static_cast<const T *>(p.branch) + row * p.sb, p, at.lane, b);
        if (p.gate) load_row<V, E>(static_cast<const T *>(p.gate) + row * p.sg, p, at.lane, a);
        if (g_out) {
            load_row<V, E>(g_out + row * sgo, p, at.lane, gx);
        } else {
#pragma unroll
            for (int k = 0; k < N; ++k) gx[k] = 0.0f;
        }
        const float inv_y = inv[2 * row], inv_x = inv[2 * row + 1];
        float unit[N];  // y^
        if (p.branch) {
#pragma unroll
            for (int k = 0; k < N; ++k) {
                unit[k] = b[k] * inv_y;
                if (p.gate) unit[k] *= a[k] * sigmoid_fast(a[k]);
                x[k] = fmaf(both[k], unit[k], x[k]);
            }
        }
        if (g_next) {
            float v[N], sum = 0.0f;
            load_row<V, E>(g_next + row * sgn, p, at.lane, v);
#pragma unroll
            for (int k = 0; k < N; ++k) {
                x[k] *= inv_x;  // x'^
                if (there) sum_next[k] = fmaf(v[k], x[k], sum_next[k]);
                v[k] *= next[k];
                sum = fmaf(v[k], x[k], sum);
            }
            const float mean = row_sum(sum) * share;
#pragma unroll
            for (int k = 0; k < N; ++k) gx[k] = fmaf(inv_x, fmaf(-x[k], mean, v[k]), gx[k]);
        }
        if (g_x && there) store_row<V, E>(g_x + row * p.channels, p, at.lane, gx);
        if (!p.branch) continue;
        float sum = 0.0f;
#pragma unroll
        for (int k = 0; k < N; ++k) {
            if (there) sum_both[k] = fmaf(gx[k], unit[k], sum_both[k]);
            gx[k] *= both[k];
            sum = fmaf(gx[k], unit[k], sum);
        }
        const float mean = row_sum(sum) * share;
#pragma unroll
        for (int k = 0; k < N; ++k) gx[k] = inv_y * fmaf(-unit[k], mean, gx[k]);  // gy
        if (p.gate) {
            float dgate[N];
#pragma unroll
            for (int k = 0; k < N; ++k) {
                const float sig = sigmoid_fast(a[k]);
                dgate[k] = gx[k] * b[k] * sig * fmaf(a[k], 1.0f - sig, 1.0f);
                gx[k] *= a[k] * sig;
            }
            if (g_gate && there) store_row<V, E>(g_gate + row * p.channels, p, at.lane, dgate);
        }
        if (g_branch && there) store_row<V, E>(g_branch + row * p.channels, p, at.lane, gx);
    }
    // the groups of the workgroup one after another
    float *out = part + int64_t(blockIdx.x) * 2 * p.channels;
    for (int g = 0; g < at.groups; ++g) {
        if (at.group == g) {
            each_channel<V, E, N>(p, at.lane, [&](int c, int k) {
                float both_c = sum_both[k], next_c = sum_next[k];
                if (g > 0) {
                    both_c += sums[c];
                    next_c += sums[p.channels + c];
                }
                if (g == at.groups - 1) {
                    out[c] = both_c;
                    out[p.channels + c] = next_c;
                } else {
                    sums[c] = both_c;
                    sums[p.channels + c] = next_c;
                }
            });
        }
        if (g < at.groups - 1) __syncthreads();
    }
}

// the weights' gradients (NULL: not asked for) from the partial sums: blockIdx.y 0
// post and scale, 1 next
__global__ void __launch_bounds__(kSumShares *kSumColumns)
    residual_norm_sum_kernel(const float *part, int64_t parts, int64_t channels, const float *post,
                             const float *scale, float *g_post, float *g_scale, float *g_next) {
    if (blockIdx.y == 1 ? !g_next : !g_post && !g_scale) return;
    const int64_t c = int64_t(blockIdx.x) * kSumColumns + threadIdx.x % kSumColumns;
    const float sum = sum_parts(part + blockIdx.y * channels, parts, 2 * channels, c, channels);
    if (threadIdx.x >= kSumColumns || c >= channels) return;
    if (blockIdx.y == 1) {
        g_next[c] = sum;
    } else {
        if (g_post) g_post[c] = sum * (scale ? scale[c] : 1.0f);
        if (g_scale) g_scale[c] = sum * post[c];
    }
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

// How rows are spread.  elements: of a thread; lanes: of a row, the fewest of a
// power of two; whole: channels in whole 16 byte moves of the branch's type.
//
// The forward takes 16 elements above 512 channels, so that rows of up to 1024
// stay in one wavefront and need no barrier: 60016 x 1024 (bfloat16 under a
// float32 stream) 162 us, against 191 us with 8.  The backward holds twice as
// much and takes 8 up to 4096 channels (a quarter of a SIMD's registers per
// wavefront then, half with 16): 259 us, against 296 us with 16; 9000 x 3104
// bfloat16 with the forward 219 us, against 262 us.
struct NormPlan {
    int elements, lanes, threads, whole;
    int64_t passes(int64_t rows) const { return cdiv(rows, threads / lanes); }
};

constexpr int64_t kFwdWorkgroups = 2048, kBwdWorkgroups = 1024;
constexpr int kFwdNarrow = 8 * kWave, kBwdNarrow = 64 * kWave;

static int64_t fwd_workgroups(int64_t passes) { return passes < kFwdWorkgroups ? passes : kFwdWorkgroups; }

// At least two rows each, where there are: partial sums are written and read
// for every workgroup (4008 x 512: their sum 6.6 -> 4.0 us, the rest unchanged).
static int64_t bwd_workgroups(int64_t passes) {
    const int64_t half = cdiv(passes, 2);
    return half < kBwdWorkgroups ? half : kBwdWorkgroups;
}

static NormPlan norm_plan(const pesq_residual_norm *p, int narrow) {
    NormPlan plan;
    plan.elements = p->channels <= narrow ? 8 : 16;
    plan.lanes = plan.elements == 8 ? 16 : kWave;
    plan.whole = static_cast<int>(p->channels / (16 / type_size(p->dtype)) * (16 / type_size(p->dtype)));
    while (plan.lanes * plan.elements < plan.whole) plan.lanes *= 2;
    plan.threads = plan.lanes > kNormThreads ? plan.lanes : kNormThreads;
    return plan;
}

static NormArgs norm_args(const pesq_residual_norm *p, const NormPlan &plan) {
    return {p->rows, p->channels, p->x, p->branch, p->gate, p->strides[0], p->strides[1],
            p->strides[2], p->post_weight, p->scale, p->next_weight, static_cast<float>(p->eps), plan.lanes,
            plan.whole};
}

// fn(V, E, width, tail) as constants
template <class T, class Fn>
static void with_plan(const NormPlan &plan, bool tail, Fn fn) {
    using std::integral_constant;
    const integral_constant<int, 16 / sizeof(T)> v;
    const auto with_tail = [&](auto e, auto width) {
        if (tail) {
            fn(v, e, width, std::true_type());
        } else {
            fn(v, e, width, std::false_type());
        }
    };
    const integral_constant<int, 8> e;
    if (plan.elements == 16) return with_tail(integral_constant<int, 16>(), integral_constant<int, 64>());
    if (plan.lanes == 16) return with_tail(e, integral_constant<int, 16>());
    if (plan.lanes == 32) return with_tail(e, integral_constant<int, 32>());
    with_tail(e, integral_constant<int, 64>());
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
    *backward = size_t(bwd_workgroups(p->rows)) * 2 * p->channels * sizeof(float);
    return PESQ_OK;
}

extern "C" int pesq_residual_norm_forward(const pesq_residual_norm *p, void *x_out, void *n_out,
                                          float *inverse, hipStream_t stream) {
    if (int st = check_norm_operands(p)) return st;
    if (p->rows == 0) return PESQ_OK;
    PESQ_CHECK_ARG((!p->branch || x_out) && (!p->next_weight || n_out), "null argument");
    const NormPlan plan = norm_plan(p, kFwdNarrow);
    const unsigned grid = static_cast<unsigned>(fwd_workgroups(plan.passes(p->rows)));
    with_types(p, [&](auto s, auto t) {
        using S = decltype(s);
        using T = decltype(t);
        with_plan<T>(plan, plan.whole < p->channels, [&](auto v, auto e, auto width, auto tail) {
            residual_norm_fwd_kernel<S, T, v.value, e.value, width.value, tail.value>
                <<<grid, plan.threads, 0, stream>>>(
                    norm_args(p, plan), static_cast<S *>(x_out), static_cast<T *>(n_out), inverse);
        });
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
    PESQ_CHECK_ARG(!g_next || g_n_out || p->rows == 0, "the next weight's gradient without n's");
    PESQ_CHECK_ARG(!g_scale || p->post_weight, "null argument");
    const int64_t channels = p->channels;
    const NormPlan plan = norm_plan(p, kBwdNarrow);
    float *part = static_cast<float *>(workspace);
    const int64_t parts = bwd_workgroups(plan.passes(p->rows));
    if (p->rows > 0) {
        with_types(p, [&](auto s, auto t) {
            using S = decltype(s);
            using T = decltype(t);
            with_plan<T>(plan, plan.whole < p->channels, [&](auto v, auto e, auto width, auto tail) {
                residual_norm_bwd_kernel<S, T, v.value, e.value, width.value, tail.value>
                    <<<static_cast<unsigned>(parts), plan.threads, 0, stream>>>(
                        norm_args(p, plan), static_cast<const S *>(g_x_out), g_strides[0],
                        static_cast<const T *>(g_n_out), g_strides[1], inverse, static_cast<S *>(g_x),
                        static_cast<T *>(g_branch), static_cast<T *>(g_gate), part);
            });
        });
        PESQ_CHECK_LAUNCH("pesq_residual_norm_backward");
    }
    if (g_post || g_scale || g_next) {
        residual_norm_sum_kernel<<<dim3(static_cast<unsigned>(cdiv(channels, kSumColumns)), 2),
                                   kSumShares * kSumColumns, 0, stream>>>(
            part, parts, channels, p->post_weight, p->scale, g_post, g_scale, g_next);
        PESQ_CHECK_LAUNCH("pesq_residual_norm_backward");
    }
    return PESQ_OK;
}
