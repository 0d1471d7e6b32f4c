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
//   2. the pairs of the chunk are joined and published; those of the chunks before
//      it are read (each wavefront's first look is made with its inputs, so most
//      have arrived by then) and folded, from the initial state on, into the state
//      at the chunk's start;
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

constexpr int kSteps = 8;           // of a wavefront, and between two kept states
constexpr int kWaves = 8;           // of a workgroup,
constexpr int kMaxWaves = 16;       // and of one of a long row
constexpr int kLongRow = 256;       // chunks of kWaves parts from which a row is long
constexpr int kFan = 16;            // chunks whose pairs are joined into one
constexpr int kRound = 16;          // pairs folded between two barriers
constexpr int kEarly = 2;           // pairs a wavefront looks at with its inputs
constexpr int kCounters = 64;       // that rows share
constexpr int kCounterStride = 16;  // words between them: a cache line each
constexpr int kRecThreads = 64;     // of the element-wise kernels
constexpr uint64_t kPending = ~uint64_t(0);
constexpr int kPolls = 1 << 22;  // seconds, far beyond any wait: the result is NaN then

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

// V neighbouring channels of type T
template <class T, int V>
struct alignas(sizeof(T) * V) Elements {
    T v[V];
};

// Rows are moved by buffer instructions: one descriptor for a tensor's rows of a
// part, a uniform offset for the row and one register for the lane's, which is
// past every buffer's end (reads zeros, writes nothing) for a lane past the
// row's.
using Buffer = __amdgpu_buffer_rsrc_t;
constexpr int kBufferBytes = 0x7fffffff;
constexpr uint32_t kNoLane = 0x80000000u;

// (none of it is there if p is null)
__device__ __forceinline__ Buffer buffer_of(const void *p, bool there) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<void *>(p), 0, there ? kBufferBytes : 0, 0x00020000);
}

// element: the lane's first one, or kNoLane
template <class T, int V>
__device__ __forceinline__ Elements<T, V> load_elements(Buffer buffer, uint32_t element, int row) {
    using E = Elements<T, V>;
    const int offset = static_cast<int>(element == kNoLane ? kNoLane : element * sizeof(T));
    if constexpr (sizeof(E) == 2) {
        return __builtin_bit_cast(E, __builtin_amdgcn_raw_buffer_load_b16(buffer, offset, row, 0));
    } else if constexpr (sizeof(E) == 4) {
        return __builtin_bit_cast(E, __builtin_amdgcn_raw_buffer_load_b32(buffer, offset, row, 0));
    } else if constexpr (sizeof(E) == 8) {
        return __builtin_bit_cast(E, __builtin_amdgcn_raw_buffer_load_b64(buffer, offset, row, 0));
    } else {
        return __builtin_bit_cast(E, __builtin_amdgcn_raw_buffer_load_b128(buffer, offset, row, 0));
    }
}

template <class T, int V>
__device__ __forceinline__ void store_elements(Buffer buffer, uint32_t element, int row, const float (&f)[V]) {
    using E = Elements<T, V>;
    E e;
#pragma unroll
    for (int k = 0; k < V; ++k) e.v[k] = static_cast<T>(f[k]);
    const int offset = static_cast<int>(element == kNoLane ? kNoLane : element * sizeof(T));
    if constexpr (sizeof(E) == 2) {
        __builtin_amdgcn_raw_buffer_store_b16(__builtin_bit_cast(uint16_t, e), buffer, offset, row, 0);
    } else if constexpr (sizeof(E) == 4) {
        __builtin_amdgcn_raw_buffer_store_b32(__builtin_bit_cast(uint32_t, e), buffer, offset, row, 0);
    } else if constexpr (sizeof(E) == 8) {
        typedef uint32_t __attribute__((ext_vector_type(2))) Words;
        __builtin_amdgcn_raw_buffer_store_b64(__builtin_bit_cast(Words, e), buffer, offset, row, 0);
    } else {
        typedef uint32_t __attribute__((ext_vector_type(4))) Words;
        __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(Words, e), buffer, offset, row, 0);
    }
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

// A chunk: its number in the order of the fold, batch item and channels
struct Place {
    int64_t chunk, row, b;
    int c0;            // first channel of the group
    uint32_t element;  // the lane's first, after it, or kNoLane
};

// LDS of a workgroup: its parts' pairs, those of earlier chunks, and the state
// before the chunk
template <int V>
struct Shared {
    Pair parts[kMaxWaves][V][kWave];
    Pair words[kRound][V][kWave];
    float heads[V][kWave];
    uint32_t ticket;
};

__device__ __forceinline__ uint64_t look(const uint64_t *word) {
    return __hip_atomic_load(word, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

// A word once it is there, from the first look at it on
__device__ __forceinline__ Pair wait_for(const uint64_t *word, uint64_t got) {
    for (int poll = 0; poll < kPolls && got == kPending; ++poll) got = look(word);
    return {__uint_as_float(static_cast<uint32_t>(got)), __uint_as_float(static_cast<uint32_t>(got >> 32))};
}

// A workgroup's chunk: rows (batch items times channel groups) go by the
// workgroup's number, and the chunk is the next one of the row in the order of
// the fold, by a counter (from kPending on) of kCounters that rows share.
template <int V>
__device__ __forceinline__ Place place_of(const RecArgs &p, uint64_t *words, int lane, Shared<V> &lds) {
    const uint32_t rows = static_cast<uint32_t>(p.batch) * p.groups;
    const uint32_t lanes = rows < kCounters ? rows : kCounters;
    // (every lane gets as many workgroups as its rows have chunks)
    const uint32_t own = blockIdx.x % rows % lanes, count = (rows - own + lanes - 1) / lanes;
    uint32_t ticket = blockIdx.x / lanes;
    if (p.chunks > 1) {
        if (threadIdx.x == 0) {
            lds.ticket = static_cast<uint32_t>(__hip_atomic_fetch_add(words + own * kCounterStride, uint64_t(1),
                                                                      __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) + 1);
        }
        __syncthreads();
        ticket = lds.ticket;
    }
    // (divisions leave uniform values in vector registers)
    ticket = __builtin_amdgcn_readfirstlane(ticket);
    const uint32_t chunk = __builtin_amdgcn_readfirstlane(ticket / count);
    const uint32_t row = own + lanes * (ticket - chunk * count);
    const int b = __builtin_amdgcn_readfirstlane(static_cast<int>(row / p.groups));
    Place at;
    at.chunk = chunk;
    at.row = row;
    at.b = b;
    at.c0 = __builtin_amdgcn_readfirstlane((static_cast<int>(row) - b * p.groups) * kWave * V);
    at.element = lane * V < static_cast<int>(p.channels) - at.c0 ? lane * V : kNoLane;
    return at;
}

// The published pairs of a row: of its chunks, and of kFan chunks each.
// words: counters, then [chunks][rows][V][64], then [chunks / kFan][rows][V][64]
template <int V>
struct Published {
    uint64_t *pairs, *joined;  // of this row and lane
    int64_t stride;            // to the next chunk's
    int64_t fan, in_fan;       // joined ones before this chunk, and chunks after them
    int64_t items, first;      // to fold: in_fan pairs, then the joined ones; of these, in the first round

    __device__ __forceinline__ Published(const RecArgs &p, const Place &at, uint64_t *words, int lane) {
        stride = p.batch * p.groups * (V * kWave);
        pairs = words + kCounters * kCounterStride + at.row * (V * kWave) + lane;
        joined = pairs + p.chunks * stride;
        fan = p.chunks > 1 ? at.chunk / kFan : 0;
        in_fan = p.chunks > 1 ? at.chunk % kFan : 0;
        items = fan + in_fan;
        // the pairs alone, where others wait for their joined one
        first = in_fan == kFan - 1 ? in_fan : items < kRound ? items : kRound;
    }
    __device__ __forceinline__ const uint64_t *item(int64_t k) const {
        return k < in_fan ? pairs + (fan * kFan + k) * stride : joined + (k - in_fan) * stride;
    }
};

// Each wavefront's first look at a word, together with its inputs: most are there
template <int V>
struct Early {
    uint64_t got[kEarly][V];
    __device__ __forceinline__ void load(const Published<V> &of, int wave, int waves) {
#pragma unroll
        for (int n = 0; n < kEarly; ++n) {
            const int64_t k = wave + n * waves;
#pragma unroll
            for (int v = 0; v < V; ++v) got[n][v] = k < of.first ? look(of.item(k) + v * kWave) : kPending;
        }
    }
};

// The state before this chunk into lds.heads, from the one before all (initial)
// and the pairs of the chunks before it; publishes this chunk's pair, and for
// the last of kFan chunks that of all of them.  The parts' pairs are in LDS; the
// wavefronts wait for some words each, and wavefront v (all of them, in turn, if
// there are fewer) folds channel v of each lane.
template <int V, bool kBack>
__device__ __forceinline__ void join_chunks(const RecArgs &p, const Place &at, const Published<V> &of,
                                            const Early<V> &early, int lane, int wave, int waves,
                                            const Elements<float, V> &initial, Shared<V> &lds) {
    Pair own[V], near[V];
    float h[V];
#pragma unroll
    for (int v = 0; v < V; ++v) {
        if (v % waves != wave) continue;
        h[v] = initial.v[v];
        near[v] = {1.0f, 0.0f};
        if (p.chunks == 1) continue;
        own[v] = lds.parts[kBack ? waves - 1 : 0][v][lane];
        for (int w = 1; w < waves; ++w) own[v] = own[v].then(lds.parts[kBack ? waves - 1 - w : w][v][lane]);
        publish(of.pairs + at.chunk * of.stride + v * kWave, own[v]);
    }
    for (int64_t first = 0; first < of.items;) {
        const int64_t left = first == 0 ? of.first : of.items - first;
        const int here = static_cast<int>(left < kRound ? left : kRound);
        for (int k = wave, n = 0; k < here; k += waves, ++n) {
            const uint64_t *word = of.item(first + k);
#pragma unroll
            for (int v = 0; v < V; ++v) {
                uint64_t got = kPending;
                if (first == 0) {
#pragma unroll
                    for (int m = 0; m < kEarly; ++m) got = n == m ? early.got[m][v] : got;
                }
                lds.words[k][v][lane] = wait_for(word + v * kWave, got);
            }
        }
        __syncthreads();
#pragma unroll
        for (int v = 0; v < V; ++v) {
            if (v % waves != wave) continue;
            for (int k = 0; k < here; ++k) {
                const Pair q = lds.words[k][v][lane];
                if (first + k < of.in_fan) {
                    near[v] = near[v].then(q);
                } else {
                    h[v] = q(h[v]);
                }
            }
            if (first == 0 && of.in_fan == kFan - 1) {
                publish(of.joined + of.fan * of.stride + v * kWave, near[v].then(own[v]));
            }
        }
        first += here;
        if (first < of.items) __syncthreads();
    }
#pragma unroll
    for (int v = 0; v < V; ++v) {
        if (v % waves == wave) lds.heads[v][lane] = near[v](h[v]);
    }
    __syncthreads();
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

// The rows of a wavefront's steps n0 .. n0 + steps - 1 of one tensor, one after
// another; after the last step, that one again.
struct Rows {
    Buffer buffer;
    int offset, stride, left;  // in bytes; steps still to come after this one
    __device__ __forceinline__ int next() {
        const int row = offset;
        offset += left > 0 ? stride : 0;
        --left;
        return row;
    }
};

template <class T>
__device__ __forceinline__ Rows rows_of(const RecArgs &p, const Place &at, int64_t n0, int steps,
                                        const void *tensor, int64_t sb, int64_t st) {
    const int64_t t = p.reverse ? p.time - n0 - steps : n0, size = sizeof(T);
    const int stride = static_cast<int>(st * size);
    return {buffer_of(static_cast<const char *>(tensor) + (at.b * sb + t * st + at.c0) * size, tensor),
            p.reverse ? (steps - 1) * stride : 0, p.reverse ? -stride : stride, steps - 1};
}

// What a wavefront's part of a chunk needs from memory, requested all at once.
// (steps past the end stand for the last one; none of an empty part)
template <class T, int V, bool kReset, int kTensors>
struct Part {
    Elements<T, V> e[kTensors][kSteps];  // r, i, x and, backward, dy
    Elements<float, V> decay, start, initial;
    uint32_t resets;
    int64_t n0;
    int left;

    __device__ __forceinline__ void load(const RecArgs &p, const Place &at, int64_t n, int lane, const void *gy,
                                         int64_t sgb, int64_t sgt, const float *starts, const float *first) {
        n0 = n;
        left = n0 >= p.time ? 0 : p.time - n0 < kSteps ? static_cast<int>(p.time - n0) : kSteps;
        if (left > 0) {
            Rows r = rows_of<T>(p, at, n0, left, p.r, p.srb, p.srt);
            Rows i = rows_of<T>(p, at, n0, left, p.i, p.sib, p.sit);
            Rows x = rows_of<T>(p, at, n0, left, p.x, p.sxb, p.sxt);
#pragma unroll
            for (int s = 0; s < kSteps; ++s) {
                e[0][s] = load_elements<T, V>(r.buffer, at.element, r.next());
                e[1][s] = load_elements<T, V>(i.buffer, at.element, i.next());
                e[2][s] = load_elements<T, V>(x.buffer, at.element, x.next());
            }
            if constexpr (kTensors == 4) {
                Rows g = rows_of<T>(p, at, n0, left, gy, sgb, sgt);
#pragma unroll
                for (int s = 0; s < kSteps; ++s) {
                    e[3][s] = load_elements<T, V>(g.buffer, at.element, g.next());
                }
            }
        }
        if constexpr (kTensors == 4) {
            const float *from = starts + (at.b * cdiv(p.time, kSteps) + n0 / kSteps) * p.channels + at.c0;
            start = load_elements<float, V>(buffer_of(from, left > 0), at.element, 0);
        }
        initial = load_elements<float, V>(buffer_of(first + at.b * p.channels + at.c0, first), at.element, 0);
        decay = load_elements<float, V>(buffer_of(p.decay + at.c0, true), at.element, 0);
        resets = reset_bits<kReset>(p, at.b, n0, lane);
    }
};

template <class T, int V, bool kReset>
__global__ void __launch_bounds__(kMaxWaves *kWave)
    recurrence_fwd_kernel(RecArgs p, T *y, float *last, float *starts, uint64_t *words) {
    __shared__ Shared<V> lds;
    const int lane = lane_id(), wave = wave_index(), waves = blockDim.x / kWave;
    const Place here = place_of<V>(p, words, lane, lds);
    Part<T, V, kReset, 3> part;
    part.load(p, here, (here.chunk * waves + wave) * kSteps, lane, nullptr, 0, 0, nullptr, p.initial);
    const Published<V> of(p, here, words, lane);
    Early<V> early;
    early.load(of, wave, waves);
    __builtin_amdgcn_sched_barrier(0);  // every load is on its way before the first wait
    const int left = part.left;
    const int64_t n0 = part.n0;
    const uint32_t resets = part.resets;
    Rate rate[V];
    float a[kSteps][V], in[kSteps][V], h[V];
    Pair own[V];
#pragma unroll
    for (int v = 0; v < V; ++v) {
        rate[v] = channel_rate(part.decay.v[v], p.rate);
        own[v] = {1.0f, 0.0f};
    }
    const auto steps = [&](auto full) {
#pragma unroll
        for (int s = 0; s < kSteps; ++s) {
            const bool there = full.value || s < left, drop = kReset && (resets >> s & 1);
#pragma unroll
            for (int v = 0; v < V; ++v) {
                const Gates g = gates(static_cast<float>(part.e[0][s].v[v]),
                                      static_cast<float>(part.e[1][s].v[v]), rate[v]);
                a[s][v] = there ? g.a : 1.0f;
                in[s][v] = there ? g.s * g.open_i * static_cast<float>(part.e[2][s].v[v]) : 0.0f;
                own[v].a = drop ? 0.0f : own[v].a * a[s][v];
                own[v].b = drop ? in[s][v] : fmaf(a[s][v], own[v].b, in[s][v]);
            }
        }
    };
    if (left == kSteps) {
        steps(std::true_type());
    } else if (left > 0) {
        steps(std::false_type());
    }
#pragma unroll
    for (int v = 0; v < V; ++v) lds.parts[wave][v][lane] = own[v];
    __syncthreads();
    join_chunks<V, false>(p, here, of, early, lane, wave, waves, part.initial, lds);
#pragma unroll
    for (int v = 0; v < V; ++v) {
        h[v] = lds.heads[v][lane];
        for (int w = 0; w < wave; ++w) h[v] = lds.parts[w][v][lane](h[v]);
    }
    if (left > 0) {
        const float *out = starts + (here.b * cdiv(p.time, kSteps) + n0 / kSteps) * p.channels + here.c0;
        store_elements<float, V>(buffer_of(out, starts), here.element, 0, h);
        Rows to = rows_of<T>(p, here, n0, left, y, p.time * p.channels, p.channels);
#pragma unroll
        for (int s = 0; s < kSteps; ++s) {
            const bool drop = kReset && (resets >> s & 1);
#pragma unroll
            for (int v = 0; v < V; ++v) h[v] = drop ? in[s][v] : fmaf(a[s][v], h[v], in[s][v]);
            // (a step past the end leaves h and writes the last row again)
            store_elements<T, V>(to.buffer, here.element, to.next(), h);
        }
    }
    if (last && wave == waves - 1 && here.chunk == p.chunks - 1) {
        store_elements<float, V>(buffer_of(last + here.b * p.channels + here.c0, true), here.element, 0, h);
    }
}

// G as a carry c between steps: g = dy + c, c = a g (0 at a reset), from the
// last step to the first; chunk 0 of the fold is the last in time.
template <class T, int V, bool kReset>
__global__ void __launch_bounds__(kMaxWaves *kWave)
    recurrence_bwd_kernel(RecArgs p, const T *gy, int64_t sgb, int64_t sgt, const float *g_last,
                          const float *starts, T *gx, T *gr, T *gi, float *decay_part,
                          float *g_initial, uint64_t *words) {
    __shared__ Shared<V> lds;
    __shared__ float sums[kMaxWaves][kWave][V];
    const int lane = lane_id(), wave = wave_index(), waves = blockDim.x / kWave;
    const Place here = place_of<V>(p, words, lane, lds);
    Part<T, V, kReset, 4> part;
    part.load(p, here, ((p.chunks - 1 - here.chunk) * waves + wave) * kSteps, lane, gy, sgb, sgt, starts, g_last);
    const Published<V> of(p, here, words, lane);
    Early<V> early;
    early.load(of, wave, waves);
    __builtin_amdgcn_sched_barrier(0);  // every load is on its way before the first wait
    const int left = part.left;
    const int64_t n0 = part.n0;
    const uint32_t resets = part.resets;
    Rate rate[V];
    float open_r[kSteps][V], a[kSteps][V], g[kSteps][V], c[V], sum[V], h[V];
    Elements<T, V> ri[kSteps], rx[kSteps];
    Pair own[V];
#pragma unroll
    for (int v = 0; v < V; ++v) {
        rate[v] = channel_rate(part.decay.v[v], p.rate);
        h[v] = part.start.v[v];
        sum[v] = 0.0f;
        own[v] = {1.0f, 0.0f};
    }
#pragma unroll
    for (int s = 0; s < kSteps; ++s) {
        ri[s] = part.e[1][s];
        rx[s] = part.e[2][s];
    }
    const auto towards_start = [&](auto full) {
#pragma unroll
        for (int s = kSteps - 1; s >= 0; --s) {
            const bool there = full.value || s < left, drop = kReset && (resets >> s & 1);
#pragma unroll
            for (int v = 0; v < V; ++v) {
                open_r[s][v] = sigmoid_fast(static_cast<float>(part.e[0][s].v[v]));
                a[s][v] = exp2_fast(rate[v].k * open_r[s][v]);
                g[s][v] = there ? static_cast<float>(part.e[3][s].v[v]) : 0.0f;
                const float k = there ? a[s][v] : 1.0f;
                own[v].a = drop ? 0.0f : own[v].a * k;
                own[v].b = drop ? 0.0f : k * (g[s][v] + own[v].b);
            }
        }
    };
    if (left == kSteps) {
        towards_start(std::true_type());
    } else if (left > 0) {
        towards_start(std::false_type());
    }
#pragma unroll
    for (int v = 0; v < V; ++v) lds.parts[wave][v][lane] = own[v];
    __syncthreads();
    join_chunks<V, true>(p, here, of, early, lane, wave, waves, part.initial, lds);
#pragma unroll
    for (int v = 0; v < V; ++v) {
        c[v] = lds.heads[v][lane];
        for (int w = waves - 1; w > wave; --w) c[v] = lds.parts[w][v][lane](c[v]);
    }
    const auto gradients = [&](auto full) {
#pragma unroll
        for (int s = kSteps - 1; s >= 0; --s) {
            const bool there = full.value || s < left, drop = kReset && (resets >> s & 1);
#pragma unroll
            for (int v = 0; v < V; ++v) {
                g[s][v] += c[v];
                c[v] = drop ? 0.0f : there ? a[s][v] * g[s][v] : c[v];
            }
        }
        const int64_t sb = p.time * p.channels;
        Rows to_x = rows_of<T>(p, here, n0, left, gx, sb, p.channels);
        Rows to_i = rows_of<T>(p, here, n0, left, gi, sb, p.channels);
        Rows to_r = rows_of<T>(p, here, n0, left, gr, sb, p.channels);
#pragma unroll
        for (int s = 0; s < kSteps; ++s) {
            if (!full.value && s >= left) continue;
            const bool drop = kReset && (resets >> s & 1);
            float dx[V], dr[V], di[V];
#pragma unroll
            for (int v = 0; v < V; ++v) {
                const float x = static_cast<float>(rx[s].v[v]);
                const float open_i = sigmoid_fast(static_cast<float>(ri[s].v[v]));
                const float log2a = rate[v].k * open_r[s][v];
                const float scale = input_scale(log2a, a[s][v]);
                const float before = drop ? 0.0f : h[v];
                const float grad = g[s][v], gate = scale * open_i, kept = a[s][v] * before;
                const float driven = grad * gate * x;
                // a^2 / s^2 is infinite where u is 0; times s u (1 - open) it tends to 0
                const float slope = scale > 0.0f ? a[s][v] * a[s][v] * rcp_fast(scale * scale) : 0.0f;
                const float du = fmaf(slope, driven, -kept * grad);
                dx[v] = grad * gate;
                di[v] = fmaf(-driven, open_i, driven);
                dr[v] = du * (-kLn2 * log2a) * (1.0f - open_r[s][v]);
                sum[v] = fmaf(du, open_r[s][v], sum[v]);
                h[v] = fmaf(gate, x, kept);
            }
            store_elements<T, V>(to_x.buffer, here.element, to_x.next(), dx);
            store_elements<T, V>(to_i.buffer, here.element, to_i.next(), di);
            store_elements<T, V>(to_r.buffer, here.element, to_r.next(), dr);
        }
    };
    if (left == kSteps) {
        gradients(std::true_type());
    } else if (left > 0) {
        gradients(std::false_type());
    }
    if (g_initial && wave == 0 && here.chunk == p.chunks - 1) {
        store_elements<float, V>(buffer_of(g_initial + here.b * p.channels + here.c0, true), here.element, 0, c);
    }
    // the chunk's share of ddecay
#pragma unroll
    for (int v = 0; v < V; ++v) sums[wave][lane][v] = sum[v];
    __syncthreads();
    if (wave == 0) {
#pragma unroll
        for (int v = 0; v < V; ++v) {
            for (int w = 1; w < waves; ++w) sum[v] += sums[w][lane][v];
        }
        float *out = decay_part + (here.chunk * p.batch + here.b) * p.channels + here.c0;
        store_elements<float, V>(buffer_of(out, true), here.element, 0, sum);
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

// so that the offsets of a part's rows stay below 2^31 bytes
constexpr int64_t kMostStride = int64_t(1) << 26;

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
        PESQ_CHECK_ARG(k % 2 == 0 || p->strides[k / 2][1] < kMostStride,
                       "steps are at most 2^26 elements apart, got %lld", (long long)p->strides[k / 2][1]);
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
    // more wavefronts keep the chunks of a long row few: 1 x 64000 x 65 float16 forward
    // 49 -> 46 us; fewer leave room for two workgroups on a compute unit, one of
    // which computes while the other waits: 16 x 3751 x 960 bfloat16 201 -> 161 us
    const int most = parts / kWaves > kLongRow ? kMaxWaves : kWaves;
    plan.waves = parts < most ? static_cast<int>(parts < 1 ? 1 : parts) : most;
    plan.chunks = parts < 1 ? 1 : cdiv(parts, plan.waves);
    plan.words = plan.chunks == 1 ? 0
                                  : kCounters * kCounterStride + (plan.chunks + plan.chunks / kFan) * p->batch *
                                                                     plan.groups * plan.v * kWave;
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
    const Plan plan = plan_of(p, true);  // single channels need no more
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
    PESQ_CHECK_ARG(!g_y || (g_strides && g_strides[0] >= 0 && g_strides[1] >= 0 && g_strides[1] < kMostStride),
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
