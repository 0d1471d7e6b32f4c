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
// One pass over the data.  A wavefront takes kSteps steps of 64 (or 128, two a
// lane) channels and holds them in registers; the wavefronts of a workgroup take
// consecutive parts of a chunk of time, and the chunks of one row are separate
// workgroups.  A part maps the state before it to the state after it by
// h -> A h + H; parts and chunks are joined by these pairs:
//
//   1. each wavefront works its part's pair out, and leaves it in LDS;
//   2. the first wavefront joins the pairs of the chunk and publishes the
//      chunk's, then reads those of the chunks before it and folds them, from
//      the initial state on, into the state at its chunk's start;
//   3. each wavefront folds the pairs before its own part onto that state and
//      runs its steps again, from registers.
//
// Every kFan chunks the last one also publishes the pair of all of them, so a
// chunk folds at most time / (kFan chunk) + kFan - 1 pairs, and never waits for
// another's state, only for pairs, which need none: the depth is three memory
// round trips whatever the length.  The order of the folds is fixed: results do
// not depend on which workgroup was first.
//
// A published pair is one 64 bit word, written and read by relaxed device scope
// atomics and valid by itself (kPending, which a fill kernel writes, is a NaN no
// pair has), so no fence is needed.  Chunks are given out by a counter in the
// order of time: a workgroup waits only for chunks that were given out before
// its own, whose pairs do not wait for anything, so every wait ends.
//
// The backward does the same towards earlier steps for G, and takes the states
// themselves from those that the forward keeps, in float32, before each part:
// they are neither stored step by step nor rounded.
#include <cmath>
#include <type_traits>

#include "network.hpp"

namespace pesq {

constexpr int kSteps = 16;      // steps of a wavefront, and between two kept states
constexpr int kMaxWaves = 8;    // of a workgroup
constexpr int kFan = 16;        // chunks whose pairs are joined into one
constexpr int kBatch = 8;       // pairs read at once
constexpr int kRecThreads = 64; // of the element-wise kernels
constexpr uint64_t kPending = ~uint64_t(0);
constexpr int kPolls = 1 << 22; // of seconds, far beyond any wait: the result is NaN then

struct RecArgs {
    int64_t batch, time, channels;
    const void *x, *r, *i;
    int64_t sxb, sxt, srb, srt, sib, sit;
    const float *decay, *initial;
    const uint8_t *reset;
    float rate;
    bool reverse;
    int64_t chunks;  // per row
    int32_t groups;  // of 64 (or 128) channels
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

// s = sqrt(1 - a^2), 1 - a^2 = -expm1(-w) with w = 2 u: for small w by the
// polynomial, where the difference would cancel
__device__ __forceinline__ float input_scale(float log2a, float a) {
    const float w = -2.0f * kLn2 * log2a;
    float p = kP4;
    p = fmaf(p, w, kP3);
    p = fmaf(p, w, kP2);
    p = fmaf(p, w, kP1);
    p = fmaf(p, w, kP0);
    return __builtin_amdgcn_sqrtf(w < 0.5f ? p * w : fmaf(-a, a, 1.0f));
}

__device__ __forceinline__ Gates gates(float r, float i, const Rate &c) {
    Gates g;
    g.open_r = sigmoid_fast(r);
    g.open_i = sigmoid_fast(i);
    g.log2a = c.k * g.open_r;
    g.a = exp2_fast(g.log2a);
    g.s = input_scale(g.log2a, g.a);
    return g;
}

// element (b, t, c) of a tensor with the given strides
template <class T>
__device__ __forceinline__ const T *at(const void *p, int64_t b, int64_t sb, int64_t t, int64_t st,
                                       int64_t c) {
    return static_cast<const T *>(p) + b * sb + t * st + c;
}

// V neighbouring channels of type T, as one register: float32 alone, 16 bit
// types in pairs, or alone where a pair is not aligned
template <class T, int V>
struct alignas(sizeof(T) * V) Elements {
    T v[V];
};

template <class T, int V>
__device__ __forceinline__ Elements<T, V> load_elements(const T *row, int offset) {
    return *reinterpret_cast<const Elements<T, V> *>(row + offset);
}

template <class T, int V>
__device__ __forceinline__ void store_elements(T *row, int offset, const float (&f)[V]) {
    Elements<T, V> e;
#pragma unroll
    for (int k = 0; k < V; ++k) e.v[k] = static_cast<T>(f[k]);
    *reinterpret_cast<Elements<T, V> *>(row + offset) = e;
}

// The map h -> a h + b of a stretch of steps.  a is 0 where a reset (or a decay
// beyond float32) drops what came before, whatever it is.
struct Pair {
    float a, b;
    __device__ __forceinline__ float operator()(float h) const { return a == 0.0f ? b : fmaf(a, h, b); }
    // this one, then `next`
    __device__ __forceinline__ Pair then(const Pair &next) const { return {a * next.a, next(b)}; }
};

__device__ __forceinline__ void publish(uint64_t *word, Pair p) {
    const uint32_t a = p.a == p.a ? __float_as_uint(p.a) : 0x7fc00000u;  // never kPending's bits
    __hip_atomic_store(word, (uint64_t(__float_as_uint(p.b)) << 32) | a, __ATOMIC_RELAXED,
                       __HIP_MEMORY_SCOPE_AGENT);
}

// h mapped by the pairs words[k stride], k = 0 .. count - 1, for V channels,
// each waited for; with `joined`, the map of all of them too
template <int V, bool kJoin>
__device__ __forceinline__ void fold(const uint64_t *words, int64_t count, int64_t stride,
                                     float (&h)[V], Pair (&joined)[V]) {
    for (int64_t first = 0; first < count; first += kBatch) {
        uint64_t got[kBatch][V];
        bool ready = false;
        for (int poll = 0; poll < kPolls && !ready; ++poll) {
            uint64_t all = 0;
#pragma unroll
            for (int k = 0; k < kBatch; ++k) {
                const int64_t at = first + k < count ? first + k : count - 1;
#pragma unroll
                for (int v = 0; v < V; ++v) {
                    got[k][v] = __hip_atomic_load(words + at * stride + v, __ATOMIC_RELAXED,
                                                  __HIP_MEMORY_SCOPE_AGENT);
                }
            }
            bool pending = false;
#pragma unroll
            for (int k = 0; k < kBatch; ++k) {
#pragma unroll
                for (int v = 0; v < V; ++v) pending = pending || got[k][v] == kPending;
            }
            ready = !__any(pending);
        }
#pragma unroll
        for (int k = 0; k < kBatch; ++k) {
            if (first + k >= count) break;
#pragma unroll
            for (int v = 0; v < V; ++v) {
                const Pair p{__uint_as_float(static_cast<uint32_t>(got[k][v])),
                             __uint_as_float(static_cast<uint32_t>(got[k][v] >> 32))};
                h[v] = p(h[v]);
                if (kJoin) joined[v] = joined[v].then(p);
            }
        }
    }
}

// Where a workgroup stands: its chunk in the order of the fold, batch item and
// channels, and each lane's first channel (of a lane past the end: the last
// ones, which it reads and does not write).
struct Place {
    int64_t chunk, b;
    int c0, offset;  // first channel of the group; the lane's, after it
    bool valid;
};

template <int V>
__device__ __forceinline__ Place place_of(const RecArgs &p, uint32_t ticket, int lane) {
    const uint32_t rows = static_cast<uint32_t>(p.batch) * p.groups;
    Place at;
    at.chunk = ticket / rows;
    const uint32_t rest = ticket % rows;
    at.b = rest / p.groups;
    at.c0 = static_cast<int>(rest % p.groups) * kWave * V;
    const int left = static_cast<int>(p.channels) - at.c0;
    at.valid = lane * V < left;
    at.offset = at.valid ? lane * V : left - V;
    return at;
}

// The next chunk in the order of time (words[0] counts them, from kPending on).
__device__ __forceinline__ uint32_t take_ticket(const RecArgs &p, uint64_t *words) {
    if (p.chunks == 1) return blockIdx.x;
    __shared__ uint32_t ticket;
    if (threadIdx.x == 0) {
        ticket = static_cast<uint32_t>(__hip_atomic_fetch_add(words, uint64_t(1), __ATOMIC_RELAXED,
                                                              __HIP_MEMORY_SCOPE_AGENT) + 1);
    }
    __syncthreads();
    return __builtin_amdgcn_readfirstlane(ticket);
}

// The state before this chunk from those of the chunks before it (wavefront 0):
// publishes the chunk's pair, and for every kFan chunks that of all of them.
// words: [1] pairs [chunks][batch][channels], then joined ones [chunks / kFan].
template <int V>
__device__ __forceinline__ void join_chunks(const RecArgs &p, const Place &at, uint64_t *words,
                                            const Pair (&own)[V], float (&h)[V]) {
    if (p.chunks == 1) return;
    const int64_t stride = p.batch * p.channels;
    uint64_t *pairs = words + 1 + at.b * p.channels + at.c0 + at.offset;
    uint64_t *joined = pairs + p.chunks * stride;
    const int64_t fan = at.chunk / kFan, in_fan = at.chunk % kFan;
    const bool last_of_fan = in_fan == kFan - 1;
    if (at.valid) {
#pragma unroll
        for (int v = 0; v < V; ++v) publish(pairs + at.chunk * stride + v, own[v]);
    }
    Pair all[V];
    if (last_of_fan) {
        float none[V] = {};
#pragma unroll
        for (int v = 0; v < V; ++v) all[v] = {1.0f, 0.0f};
        fold<V, true>(pairs + fan * kFan * stride, in_fan, stride, none, all);
        if (at.valid) {
#pragma unroll
            for (int v = 0; v < V; ++v) publish(joined + fan * stride + v, all[v].then(own[v]));
        }
    }
    fold<V, false>(joined, fan, stride, h, all);
    fold<V, false>(pairs + fan * kFan * stride, in_fan, stride, h, all);
}

// bits of the resets of steps n0 ..
template <bool kReset>
__device__ __forceinline__ uint32_t reset_bits(const RecArgs &p, int64_t b, int64_t n0, int lane) {
    if (!kReset) return 0;
    bool set = false;
    if (lane < kSteps && n0 + lane < p.time) {
        const int64_t n = n0 + lane;
        set = p.reset[b * p.time + (p.reverse ? p.time - 1 - n : n)] != 0;
    }
    return static_cast<uint32_t>(__ballot(set));
}

template <class T, int V, bool kReset>
__global__ void __launch_bounds__(kMaxWaves *kWave)
    recurrence_fwd_kernel(RecArgs p, T *y, float *last, float *starts, uint64_t *words) {
    __shared__ Pair pairs[kMaxWaves][kWave][V];
    __shared__ float heads[kWave][V];
    const int lane = lane_id(), wave = wave_index(), waves = blockDim.x / kWave;
    const Place at = place_of<V>(p, take_ticket(p, words), lane);
    const int64_t b = at.b, n0 = (at.chunk * waves + wave) * kSteps;
    const int64_t channel = at.c0 + at.offset;

    Elements<T, V> rr[kSteps], ri[kSteps], rx[kSteps];
    const bool some = n0 < p.time;
    const auto time_of = [&](int s) {
        const int64_t n = n0 + s < p.time ? n0 + s : p.time - 1;
        return p.reverse ? p.time - 1 - n : n;
    };
    if (some) {
#pragma unroll
        for (int s = 0; s < kSteps; ++s) {
            const int64_t t = time_of(s);
            rr[s] = load_elements<T, V>(pesq::at<T>(p.r, b, p.srb, t, p.srt, at.c0), at.offset);
            ri[s] = load_elements<T, V>(pesq::at<T>(p.i, b, p.sib, t, p.sit, at.c0), at.offset);
            rx[s] = load_elements<T, V>(pesq::at<T>(p.x, b, p.sxb, t, p.sxt, at.c0), at.offset);
        }
    }
    const uint32_t resets = reset_bits<kReset>(p, b, n0, lane);
    Rate rate[V];
#pragma unroll
    for (int v = 0; v < V; ++v) rate[v] = channel_rate(p.decay[channel + v], p.rate);

    float a[kSteps][V], in[kSteps][V];
    Pair own[V];
#pragma unroll
    for (int v = 0; v < V; ++v) own[v] = {1.0f, 0.0f};
    if (some) {
#pragma unroll
        for (int s = 0; s < kSteps; ++s) {
            const bool there = n0 + s < p.time, drop = kReset && (resets >> s & 1);
#pragma unroll
            for (int v = 0; v < V; ++v) {
                const Gates g = gates(static_cast<float>(rr[s].v[v]), static_cast<float>(ri[s].v[v]), rate[v]);
                a[s][v] = there ? g.a : 1.0f;
                in[s][v] = there ? g.s * g.open_i * static_cast<float>(rx[s].v[v]) : 0.0f;
                own[v].a = drop ? 0.0f : own[v].a * a[s][v];
                own[v].b = drop ? in[s][v] : fmaf(a[s][v], own[v].b, in[s][v]);
            }
        }
    }
#pragma unroll
    for (int v = 0; v < V; ++v) pairs[wave][lane][v] = own[v];
    __syncthreads();
    if (wave == 0) {
        float h[V];
#pragma unroll
        for (int v = 0; v < V; ++v) h[v] = p.initial ? p.initial[b * p.channels + channel + v] : 0.0f;
        Pair chunk[V];
#pragma unroll
        for (int v = 0; v < V; ++v) {
            chunk[v] = own[v];
            for (int w = 1; w < waves; ++w) chunk[v] = chunk[v].then(pairs[w][lane][v]);
        }
        join_chunks<V>(p, at, words, chunk, h);
#pragma unroll
        for (int v = 0; v < V; ++v) heads[lane][v] = h[v];
    }
    __syncthreads();
    float h[V];
#pragma unroll
    for (int v = 0; v < V; ++v) {
        h[v] = heads[lane][v];
        for (int w = 0; w < wave; ++w) h[v] = pairs[w][lane][v](h[v]);
    }
    if (some && starts && at.valid) {
        float *out = starts + (b * cdiv(p.time, kSteps) + n0 / kSteps) * p.channels + at.c0;
        store_elements<float, V>(out, at.offset, h);
    }
    if (some) {
#pragma unroll
        for (int s = 0; s < kSteps; ++s) {
            const bool drop = kReset && (resets >> s & 1);
#pragma unroll
            for (int v = 0; v < V; ++v) h[v] = drop ? in[s][v] : fmaf(a[s][v], h[v], in[s][v]);
            if (n0 + s < p.time && at.valid) {
                store_elements<T, V>(y + (b * p.time + time_of(s)) * p.channels + at.c0, at.offset, h);
            }
        }
    }
    if (last && wave == waves - 1 && at.chunk == p.chunks - 1 && at.valid) {
        store_elements<float, V>(last + b * p.channels + at.c0, at.offset, h);
    }
}

// G as a carry c between steps: g = dy + c, c = a g (0 at a reset), from the
// last step to the first; chunk 0 of the fold is the last in time.
template <class T, int V, bool kReset>
__global__ void __launch_bounds__(kMaxWaves *kWave)
    recurrence_bwd_kernel(RecArgs p, const T *gy, int64_t sgb, int64_t sgt, const float *g_last,
                          const float *starts, T *gx, T *gr, T *gi, float *decay_part,
                          float *g_initial, uint64_t *words) {
    __shared__ Pair pairs[kMaxWaves][kWave][V];
    __shared__ float heads[kWave][V];
    const int lane = lane_id(), wave = wave_index(), waves = blockDim.x / kWave;
    const Place at = place_of<V>(p, take_ticket(p, words), lane);
    const int64_t b = at.b, n0 = ((p.chunks - 1 - at.chunk) * waves + wave) * kSteps;
    const int64_t channel = at.c0 + at.offset;

    Elements<T, V> rr[kSteps], ri[kSteps], rx[kSteps], rg[kSteps];
    const bool some = n0 < p.time;
    const auto time_of = [&](int s) {
        const int64_t n = n0 + s < p.time ? n0 + s : p.time - 1;
        return p.reverse ? p.time - 1 - n : n;
    };
    float h[V];
    if (some) {
#pragma unroll
        for (int s = 0; s < kSteps; ++s) {
            const int64_t t = time_of(s);
            rr[s] = load_elements<T, V>(pesq::at<T>(p.r, b, p.srb, t, p.srt, at.c0), at.offset);
            if (gy) rg[s] = load_elements<T, V>(pesq::at<T>(gy, b, sgb, t, sgt, at.c0), at.offset);
        }
#pragma unroll
        for (int s = 0; s < kSteps; ++s) {
            const int64_t t = time_of(s);
            ri[s] = load_elements<T, V>(pesq::at<T>(p.i, b, p.sib, t, p.sit, at.c0), at.offset);
            rx[s] = load_elements<T, V>(pesq::at<T>(p.x, b, p.sxb, t, p.sxt, at.c0), at.offset);
        }
        const float *start = starts + (b * cdiv(p.time, kSteps) + n0 / kSteps) * p.channels + at.c0;
        const Elements<float, V> held = load_elements<float, V>(start, at.offset);
#pragma unroll
        for (int v = 0; v < V; ++v) h[v] = held.v[v];
    }
    const uint32_t resets = reset_bits<kReset>(p, b, n0, lane);
    Rate rate[V];
#pragma unroll
    for (int v = 0; v < V; ++v) rate[v] = channel_rate(p.decay[channel + v], p.rate);

    float open_r[kSteps][V], a[kSteps][V], g[kSteps][V];
    Pair own[V];
#pragma unroll
    for (int v = 0; v < V; ++v) own[v] = {1.0f, 0.0f};
    if (some) {
#pragma unroll
        for (int s = kSteps - 1; s >= 0; --s) {
            const bool there = n0 + s < p.time, drop = kReset && (resets >> s & 1);
#pragma unroll
            for (int v = 0; v < V; ++v) {
                open_r[s][v] = sigmoid_fast(static_cast<float>(rr[s].v[v]));
                a[s][v] = exp2_fast(rate[v].k * open_r[s][v]);
                g[s][v] = gy && there ? static_cast<float>(rg[s].v[v]) : 0.0f;
                const float k = there ? a[s][v] : 1.0f;
                own[v].a = drop ? 0.0f : own[v].a * k;
                own[v].b = drop ? 0.0f : k * (g[s][v] + own[v].b);
            }
        }
    }
#pragma unroll
    for (int v = 0; v < V; ++v) pairs[wave][lane][v] = own[v];
    __syncthreads();
    if (wave == 0) {
        float c[V];
#pragma unroll
        for (int v = 0; v < V; ++v) c[v] = g_last ? g_last[b * p.channels + channel + v] : 0.0f;
        Pair chunk[V];
#pragma unroll
        for (int v = 0; v < V; ++v) {
            chunk[v] = pairs[waves - 1][lane][v];
            for (int w = waves - 2; w >= 0; --w) chunk[v] = chunk[v].then(pairs[w][lane][v]);
        }
        join_chunks<V>(p, at, words, chunk, c);
#pragma unroll
        for (int v = 0; v < V; ++v) heads[lane][v] = c[v];
    }
    __syncthreads();
    float c[V], sum[V];
#pragma unroll
    for (int v = 0; v < V; ++v) {
        sum[v] = 0.0f;
        c[v] = heads[lane][v];
        for (int w = waves - 1; w > wave; --w) c[v] = pairs[w][lane][v](c[v]);
    }
    if (some) {
#pragma unroll
        for (int s = kSteps - 1; s >= 0; --s) {
            const bool there = n0 + s < p.time, drop = kReset && (resets >> s & 1);
#pragma unroll
            for (int v = 0; v < V; ++v) {
                g[s][v] += c[v];
                c[v] = drop ? 0.0f : there ? a[s][v] * g[s][v] : c[v];
            }
        }
#pragma unroll
        for (int s = 0; s < kSteps; ++s) {
            const bool there = n0 + s < p.time, drop = kReset && (resets >> s & 1);
            float dx[V], dr[V], di[V];
#pragma unroll
            for (int v = 0; v < V; ++v) {
                const float x = static_cast<float>(rx[s].v[v]);
                const float open_i = sigmoid_fast(static_cast<float>(ri[s].v[v]));
                const float log2a = rate[v].k * open_r[s][v];
                const float scale = input_scale(log2a, a[s][v]);
                const float before = drop ? 0.0f : h[v];
                const float driven = g[s][v] * open_i * x;
                // a^2 / s is infinite where u is 0; times u (1 - open) it tends to 0
                const float slope = scale > 0.0f ? a[s][v] * a[s][v] * rcp_fast(scale) : 0.0f;
                const float du = fmaf(slope, driven, -a[s][v] * before * g[s][v]);
                dx[v] = g[s][v] * scale * open_i;
                di[v] = driven * scale * (1.0f - open_i);
                dr[v] = du * (-kLn2 * log2a) * (1.0f - open_r[s][v]);
                sum[v] += there ? du * open_r[s][v] : 0.0f;
                h[v] = fmaf(a[s][v], before, scale * open_i * x);
            }
            if (there && at.valid) {
                const int64_t row = (b * p.time + time_of(s)) * p.channels + at.c0;
                if (gx) store_elements<T, V>(gx + row, at.offset, dx);
                if (gi) store_elements<T, V>(gi + row, at.offset, di);
                if (gr) store_elements<T, V>(gr + row, at.offset, dr);
            }
        }
    }
    if (g_initial && wave == 0 && at.chunk == p.chunks - 1 && at.valid) {
        store_elements<float, V>(g_initial + b * p.channels + at.c0, at.offset, c);
    }
    // the chunk's share of ddecay
    __shared__ float sums[kMaxWaves][kWave][V];
#pragma unroll
    for (int v = 0; v < V; ++v) sums[wave][lane][v] = sum[v];
    __syncthreads();
    if (wave == 0 && at.valid) {
#pragma unroll
        for (int v = 0; v < V; ++v) {
            for (int w = 1; w < waves; ++w) sum[v] += sums[w][lane][v];
        }
        float *out = decay_part + (at.chunk * p.batch + b) * p.channels + at.c0;
        store_elements<float, V>(out, at.offset, sum);
    }
}

// ddecay from the chunks' shares: kSumRows threads per channel, each a share of
// the rows, joined in LDS
constexpr int kSumRows = 16, kSumChannels = 64;
__global__ void __launch_bounds__(kSumRows *kSumChannels)
    recurrence_decay_kernel(const float *part, int64_t rows, int64_t channels, const float *decay,
                            float rate, float *g_decay) {
    __shared__ float sums[kSumRows][kSumChannels];
    const int lane = threadIdx.x % kSumChannels, share = threadIdx.x / kSumChannels;
    const int64_t c = int64_t(blockIdx.x) * kSumChannels + lane;
    float sum = 0.0f;
    if (c < channels) {
#pragma unroll 8
        for (int64_t k = share; k < rows; k += kSumRows) sum += part[k * channels + c];
    }
    sums[share][lane] = sum;
    __syncthreads();
    if (share != 0 || c >= channels) return;
    for (int k = 1; k < kSumRows; ++k) sum += sums[k][lane];
    g_decay[c] = sum * channel_rate(decay[c], rate).factor;
}

__global__ void __launch_bounds__(256) recurrence_fill_kernel(uint64_t *words, int64_t count) {
    for (int64_t k = int64_t(blockIdx.x) * 256 + threadIdx.x; k < count; k += int64_t(gridDim.x) * 256) {
        words[k] = kPending;
    }
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

// How a call is cut up.  V: channels a lane holds, two of a 16 bit type where
// every pair is aligned.  waves: of a workgroup.
struct Plan {
    int v, waves;
    int64_t chunks, groups, words;
};

static Plan plan_of(const pesq_recurrence *p, bool paired) {
    Plan plan;
    plan.v = paired ? 2 : 1;
    plan.groups = cdiv(p->channels, kWave * plan.v);
    const int64_t parts = cdiv(p->time, kSteps);
    plan.waves = parts < kMaxWaves ? static_cast<int>(parts < 1 ? 1 : parts) : kMaxWaves;
    plan.chunks = parts < 1 ? 1 : cdiv(parts, plan.waves);
    plan.words = plan.chunks == 1 ? 0
                                  : 1 + (plan.chunks + plan.chunks / kFan) * p->batch * p->channels;
    return plan;
}

static bool aligned_pair(const void *p) { return reinterpret_cast<uintptr_t>(p) % 4 == 0; }

// whether every 16 bit operand can be taken in pairs of channels
static bool pairs_fit(const pesq_recurrence *p, const void *g, const int64_t *g_strides,
                      const void *out0, const void *out1, const void *out2) {
    if (p->dtype == PESQ_F32 || p->channels % 2) return false;
    for (int k = 0; k < 6; ++k) {
        if (p->strides[k / 2][k % 2] % 2) return false;
    }
    for (const void *q : {p->x, p->recur_gate, p->input_gate, g, out0, out1, out2}) {
        if (!aligned_pair(q)) return false;
    }
    return !g || (g_strides[0] % 2 == 0 && g_strides[1] % 2 == 0);
}

static RecArgs kernel_args(const pesq_recurrence *p, const Plan &plan) {
    return {p->batch, p->time, p->channels, p->x, p->recur_gate, p->input_gate,
            p->strides[0][0], p->strides[0][1], p->strides[1][0], p->strides[1][1],
            p->strides[2][0], p->strides[2][1], p->decay, p->initial, p->reset,
            static_cast<float>(p->rate), p->reverse != 0, plan.chunks,
            static_cast<int32_t>(plan.groups)};
}

static int check_grid(const pesq_recurrence *p, const Plan &plan) {
    PESQ_CHECK_ARG(plan.chunks * p->batch * plan.groups < (int64_t(1) << 31),
                   "a recurrence of %lld x %lld x %lld is too large", (long long)p->batch,
                   (long long)p->time, (long long)p->channels);
    return PESQ_OK;
}

// fn(T(), V, reset) with V and reset as constants
template <class Fn>
static void with_variant(const pesq_recurrence *p, const Plan &plan, Fn fn) {
    const auto with_reset = [&](auto type, auto v) {
        if (p->reset) {
            fn(type, v, std::true_type());
        } else {
            fn(type, v, std::false_type());
        }
    };
    with_type(p->dtype, [&](auto type) {
        if constexpr (sizeof(type) == 2) {
            if (plan.v == 2) return with_reset(type, std::integral_constant<int, 2>());
        }
        with_reset(type, std::integral_constant<int, 1>());
    });
}

static void fill_words(const Plan &plan, uint64_t *words, hipStream_t stream) {
    if (plan.words == 0) return;
    const int64_t blocks = cdiv(plan.words, 1024);
    recurrence_fill_kernel<<<static_cast<unsigned>(blocks < 2048 ? blocks : 2048), 256, 0, stream>>>(
        words, plan.words);
}

static unsigned grid_of(const pesq_recurrence *p, const Plan &plan) {
    return static_cast<unsigned>(plan.chunks * p->batch * plan.groups);
}

}  // namespace pesq

using namespace pesq;

extern "C" int pesq_recurrence_workspace(const pesq_recurrence *p, size_t *starts, size_t *forward,
                                         size_t *backward) {
    if (int st = check_recurrence(p)) return st;
    const size_t states = size_t(p->batch) * p->channels * sizeof(float);
    const Plan plan = plan_of(p, false);  // the same for pairs of channels
    if (starts) *starts = states * cdiv(p->time, kSteps);
    if (forward) *forward = plan.words * sizeof(uint64_t);
    if (backward) *backward = plan.words * sizeof(uint64_t) + states * plan.chunks;
    return PESQ_OK;
}

extern "C" int pesq_recurrence_forward(const pesq_recurrence *p, void *y, float *last,
                                       float *starts, void *workspace, hipStream_t stream) {
    if (int st = check_operands(p)) return st;
    if (empty(p)) return PESQ_OK;
    PESQ_CHECK_ARG(y || p->time == 0, "null argument");
    const Plan plan = plan_of(p, pairs_fit(p, nullptr, nullptr, y, nullptr, nullptr));
    if (int st = check_grid(p, plan)) return st;
    PESQ_CHECK_ARG(workspace || plan.words == 0, "null argument");
    uint64_t *words = static_cast<uint64_t *>(workspace);
    fill_words(plan, words, stream);
    with_variant(p, plan, [&](auto type, auto v, auto reset) {
        using T = decltype(type);
        recurrence_fwd_kernel<T, v.value, reset.value>
            <<<grid_of(p, plan), plan.waves * kWave, 0, stream>>>(
                kernel_args(p, plan), static_cast<T *>(y), last, starts, words);
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
    PESQ_CHECK_ARG(!g_decay || p->decay, "null argument");
    const Plan plan = plan_of(p, pairs_fit(p, g_y, g_strides, g_x, g_recur, g_input));
    if (int st = check_grid(p, plan)) return st;
    uint64_t *words = static_cast<uint64_t *>(workspace);
    float *part = reinterpret_cast<float *>(words + plan.words);
    if (p->batch > 0) {
        fill_words(plan, words, stream);
        with_variant(p, plan, [&](auto type, auto v, auto reset) {
            using T = decltype(type);
            recurrence_bwd_kernel<T, v.value, reset.value>
                <<<grid_of(p, plan), plan.waves * kWave, 0, stream>>>(
                    kernel_args(p, plan), static_cast<const T *>(g_y), g_y ? g_strides[0] : 0,
                    g_y ? g_strides[1] : 0, g_last, starts, static_cast<T *>(g_x),
                    static_cast<T *>(g_recur), static_cast<T *>(g_input), part, g_initial, words);
        });
        PESQ_CHECK_LAUNCH("pesq_recurrence_backward");
    }
    if (g_decay) {
        recurrence_decay_kernel<<<static_cast<unsigned>(cdiv(p->channels, kSumChannels)),
                                  kSumRows * kSumChannels, 0, stream>>>(
            part, plan.chunks * p->batch, p->channels, p->decay, static_cast<float>(p->rate), g_decay);
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
        const dim3 grid(static_cast<unsigned>(cdiv(p->channels, kRecThreads)),
                        static_cast<unsigned>(p->batch));
        recurrence_step_kernel<T><<<grid, kRecThreads, 0, stream>>>(kernel_args(p, Plan{}), state,
                                                                    static_cast<T *>(y));
    });
    PESQ_CHECK_LAUNCH("pesq_recurrence_step");
    return PESQ_OK;
}
