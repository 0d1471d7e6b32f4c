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
// One pass over the data.  A wavefront takes kSteps steps of 64 channels and holds
// them in registers; the wavefronts of a workgroup take
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
// chunk folds at most time / (kFan chunk) + kFan - 1 pairs, kRound between two
// barriers, and never waits for another's state, only for pairs, which need none:
// three memory round trips deep however long the row, while the pairs to fold grow
// with it (64000 steps: 250 chunks, 30 pairs for the last one).  The order of the
// folds is fixed: results do not depend on which workgroup was first.
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
#include <cfloat>
#include <cmath>
#include <type_traits>

#include "network.hpp"

namespace pesq {

constexpr int kSteps = 16;          // of a wavefront, and between two kept states
constexpr int kWaves = 4;           // of a workgroup,
constexpr int kMaxWaves = 16;       // and of one of a long row
constexpr int kLongRow = 256;       // chunks of kWaves parts that a row has at most, or is long
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
    int32_t groups;  // of 64 channels
    const float *rates;  // open_log2 of every channel, or NULL
};

// log2 of a channel's a at an open gate, -rate softplus(decay) log2(e) <= 0, to
// the last bits, since its error acts on every step:
// softplus(d) = max(d, 0) + log(1 + y), y = exp(-|d|).  The exponential's argument
// is carried in two parts; log(1 + y) = 2 artanh(z), z = y / (2 + y) <= 1/3, by
// its series up to z^15.  Finite for every decay but NaN, which stays one: a gate
// that is shut (sigmoid 0) keeps the state whatever the decay.
__device__ __forceinline__ float open_log2(float decay, float rate) {
    constexpr float kLog2eRest = 1.92596299e-8f;  // log2(e) = kLog2e + this
    const float d = fminf(fabsf(decay), 128.0f), x = kLog2e * d;  // (y is 0 from 104 on)
    const float rest = fmaf(kLog2e, d, -x) + kLog2eRest * d;
    float y = exp2_fast(-x);
    y = fmaf(-kLn2 * rest, y, y);
    const float w = 2.0f + y;
    float r = rcp_fast(w);
    r = fmaf(fmaf(-w, r, 1.0f), r, r);
    const float z = y * r, t = z * z;
    float p = 1.0f / 15.0f;
    p = fmaf(p, t, 1.0f / 13.0f);
    p = fmaf(p, t, 1.0f / 11.0f);
    p = fmaf(p, t, 1.0f / 9.0f);
    p = fmaf(p, t, 1.0f / 7.0f);
    p = fmaf(p, t, 1.0f / 5.0f);
    p = fmaf(p, t, 1.0f / 3.0f);
    p = fmaf(p * t, z, z);
    const float softplus = fmaf(2.0f, p, decay < 0.0f ? 0.0f : decay), k = -softplus * (rate * kLog2e);
    return k < -FLT_MAX ? -FLT_MAX : k;
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

// k: open_log2 of the channel
__device__ __forceinline__ Gates gates(float r, float i, float k) {
    Gates g;
    g.open_r = sigmoid_fast(r);
    g.open_i = sigmoid_fast(i);
    g.log2a = k * g.open_r;
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

// Rows are moved by buffer instructions: one descriptor for a tensor's rows of a
// part, a uniform offset for the row and one register for the lane's channel,
// which is past every buffer's end (reads zeros, writes nothing) for a lane past
// the row's.
using Buffer = __amdgpu_buffer_rsrc_t;
constexpr int kBufferBytes = 0x7fffffff;
constexpr uint32_t kNoLane = 0x80000000u;

// (none of it is there if p is null)
__device__ __forceinline__ Buffer buffer_of(const void *p, bool there) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<void *>(p), 0, there ? kBufferBytes : 0, 0x00020000);
}

// channel: the lane's, from the buffer's start, or kNoLane; row: in bytes
template <class T>
__device__ __forceinline__ T load_channel(Buffer buffer, uint32_t channel, int row) {
    const int offset = static_cast<int>(channel == kNoLane ? kNoLane : channel * sizeof(T));
    if constexpr (sizeof(T) == 2) {
        return __builtin_bit_cast(T, __builtin_amdgcn_raw_buffer_load_b16(buffer, offset, row, 0));
    } else {
        return __builtin_bit_cast(T, __builtin_amdgcn_raw_buffer_load_b32(buffer, offset, row, 0));
    }
}

template <class T>
__device__ __forceinline__ void store_channel(Buffer buffer, uint32_t channel, int row, float f) {
    const int offset = static_cast<int>(channel == kNoLane ? kNoLane : channel * sizeof(T));
    const T t = static_cast<T>(f);
    if constexpr (sizeof(T) == 2) {
        __builtin_amdgcn_raw_buffer_store_b16(__builtin_bit_cast(uint16_t, t), buffer, offset, row, 0);
    } else {
        __builtin_amdgcn_raw_buffer_store_b32(__builtin_bit_cast(uint32_t, t), buffer, offset, row, 0);
    }
}

// The map h -> a h + b of a stretch of steps.  a is -0 where a reset drops what
// came before, whatever it is.  Any other a is +0 at least, a product that became
// 0 over many steps too: a NaN or an infinite h is not finite after it either, as
// step by step.
struct Pair {
    float a, b;
    // kReset: whether there are resets at all
    template <bool kReset>
    __device__ __forceinline__ bool drops() const {
        return kReset && __float_as_uint(a) == 0x80000000u;
    }
    template <bool kReset>
    __device__ __forceinline__ float after(float h) const {
        return drops<kReset>() ? b : fmaf(a, h, b);
    }
    // this one, then `next`
    template <bool kReset>
    __device__ __forceinline__ Pair then(const Pair &next) const {
        return {next.drops<kReset>() ? next.a : a * next.a, next.after<kReset>(b)};
    }
};

__device__ __forceinline__ void publish(uint64_t *word, Pair p) {
    const uint32_t a = p.a == p.a ? __float_as_uint(p.a) : 0x7fc00000u;  // never kPending's bits
    __hip_atomic_store(word, (uint64_t(__float_as_uint(p.b)) << 32) | a, __ATOMIC_RELAXED,
                       __HIP_MEMORY_SCOPE_AGENT);
}

__device__ __forceinline__ uint64_t look(const uint64_t *word) {
    return __hip_atomic_load(word, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

// A word once it is there, from the first look at it on
__device__ __forceinline__ Pair wait_for(const uint64_t *word, uint64_t got) {
    for (int poll = 0; poll < kPolls && got == kPending; ++poll) got = look(word);
    return {__uint_as_float(static_cast<uint32_t>(got)), __uint_as_float(static_cast<uint32_t>(got >> 32))};
}

// LDS of a workgroup: its parts' pairs, those of earlier chunks, and the state
// before the chunk
struct Shared {
    Pair parts[kMaxWaves][kWave];
    Pair words[kRound][kWave];
    float heads[kWave];
    uint32_t ticket;
};

// A chunk: its number in the order of the fold, row (batch item and 64 channels)
struct Place {
    int64_t chunk, row, b;
    int c0;            // first channel of the row
    uint32_t channel;  // the lane's, after it, or kNoLane
};

// A workgroup's chunk: rows go by the workgroup's number, and the chunk is the
// next one of the row in the order of the fold, by a counter (from kPending on)
// of kCounters that rows share.
__device__ __forceinline__ Place place_of(const RecArgs &p, uint64_t *words, int lane, Shared &lds) {
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
    at.c0 = __builtin_amdgcn_readfirstlane((static_cast<int>(row) - b * p.groups) * kWave);
    at.channel = lane < static_cast<int>(p.channels) - at.c0 ? lane : kNoLane;
    return at;
}

// The published pairs of a row: of its chunks, and of kFan chunks each.
// words: counters, then [chunks][rows][64], then [chunks / kFan][rows][64]
struct Published {
    uint64_t *pairs, *joined;  // of this row and lane
    int64_t stride;            // to the next chunk's
    int64_t fan, in_fan;       // joined ones before this chunk, and chunks after them
    int64_t items, first;      // to fold: in_fan pairs, then the joined ones; of these, in the first round

    __device__ __forceinline__ Published(const RecArgs &p, const Place &at, uint64_t *words, int lane) {
        stride = p.batch * p.groups * kWave;
        pairs = words + kCounters * kCounterStride + at.row * kWave + lane;
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

// Each wavefront's first look at its words, together with its inputs: most are there
struct Early {
    uint64_t got[kEarly];
    __device__ __forceinline__ void load(const Published &of, int wave, int waves) {
#pragma unroll
        for (int n = 0; n < kEarly; ++n) {
            const int64_t k = wave + n * waves;
            got[n] = k < of.first ? look(of.item(k)) : kPending;
        }
    }
};

// The state before this chunk, from the one before all (initial) and the pairs
// of the chunks before it; publishes this chunk's pair, and for the last of kFan
// chunks that of all of them.  The parts' pairs are in LDS; the wavefronts wait
// for some words each, and the first one folds them.
template <bool kBack, bool kReset>
__device__ __forceinline__ float join_chunks(const RecArgs &p, const Place &at, const Published &of,
                                             const Early &early, int lane, int wave, int waves, float initial,
                                             Shared &lds) {
    if (p.chunks == 1) return initial;
    Pair own{1.0f, 0.0f}, near{1.0f, 0.0f};
    float h = initial;
    if (wave == 0) {
        for (int w = 0; w < waves; ++w) own = own.then<kReset>(lds.parts[kBack ? waves - 1 - w : w][lane]);
        publish(of.pairs + at.chunk * of.stride, own);
    }
    for (int64_t first = 0; first < of.items;) {
        const int64_t left = first == 0 ? of.first : of.items - first;
        const int here = static_cast<int>(left < kRound ? left : kRound);
        for (int k = wave, n = 0; k < here; k += waves, ++n) {
            uint64_t got = kPending;
            if (first == 0) {
#pragma unroll
                for (int m = 0; m < kEarly; ++m) got = n == m ? early.got[m] : got;
            }
            lds.words[k][lane] = wait_for(of.item(first + k), got);
        }
        __syncthreads();
        if (wave == 0) {
            for (int k = 0; k < here; ++k) {
                const Pair q = lds.words[k][lane];
                if (first + k < of.in_fan) {
                    near = near.then<kReset>(q);
                } else {
                    h = q.after<kReset>(h);
                }
            }
            if (first == 0 && of.in_fan == kFan - 1) publish(of.joined + of.fan * of.stride, near.then<kReset>(own));
        }
        first += here;
        if (first < of.items) __syncthreads();
    }
    if (wave == 0) lds.heads[lane] = near.after<kReset>(h);
    __syncthreads();
    return lds.heads[lane];
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
template <class T, bool kReset, int kTensors>
struct Part {
    T e[kTensors][kSteps];  // r, i, x and, backward, dy
    float decay, start, initial;  // (decay: open_log2 of it where that is at hand)
    uint32_t resets;
    int left;

    __device__ __forceinline__ void load(const RecArgs &p, const Place &at, int64_t n0, int lane, const void *gy,
                                         int64_t sgb, int64_t sgt, const float *starts, const float *first) {
        left = n0 >= p.time ? 0 : p.time - n0 < kSteps ? static_cast<int>(p.time - n0) : kSteps;
        if (left > 0) {
            Rows r = rows_of<T>(p, at, n0, left, p.r, p.srb, p.srt);
            Rows i = rows_of<T>(p, at, n0, left, p.i, p.sib, p.sit);
            Rows x = rows_of<T>(p, at, n0, left, p.x, p.sxb, p.sxt);
#pragma unroll
            for (int s = 0; s < kSteps; ++s) {
                e[0][s] = load_channel<T>(r.buffer, at.channel, r.next());
                e[1][s] = load_channel<T>(i.buffer, at.channel, i.next());
                e[2][s] = load_channel<T>(x.buffer, at.channel, x.next());
            }
            if constexpr (kTensors == 4) {
                Rows g = rows_of<T>(p, at, n0, left, gy, sgb, sgt);
#pragma unroll
                for (int s = 0; s < kSteps; ++s) e[3][s] = load_channel<T>(g.buffer, at.channel, g.next());
            }
        }
        if constexpr (kTensors == 4) {
            const float *from = starts + (at.b * cdiv(p.time, kSteps) + n0 / kSteps) * p.channels + at.c0;
            start = load_channel<float>(buffer_of(from, left > 0), at.channel, 0);
        }
        initial = load_channel<float>(buffer_of(first + at.b * p.channels + at.c0, first), at.channel, 0);
        decay = load_channel<float>(buffer_of((p.rates ? p.rates : p.decay) + at.c0, true), at.channel, 0);
        resets = reset_bits<kReset>(p, at.b, n0, lane);
    }
};

// body(true or false as a constant): whether all of the part's steps are there
template <class Body>
__device__ __forceinline__ void for_part(int left, Body body) {
    if (left == kSteps) {
        body(std::true_type());
    } else if (left > 0) {
        body(std::false_type());
    }
}

// Bound by memory and by waiting: 16 x 3751 x 960 bfloat16 takes 134 us (median; 125
// to 146 by run and card), 3.5 TB/s, where the same moves alone took 103.  Five
// wavefronts a SIMD (96 registers, one spilled) hide more of the waits: 128 us against
// 142 us with the four that 97 registers leave, on one card.
template <class T, bool kReset>
__global__ void __launch_bounds__(kMaxWaves *kWave, 5)
    recurrence_fwd_kernel(RecArgs p, T *y, float *last, float *starts, uint64_t *words) {
    __shared__ Shared lds;
    const int lane = lane_id(), wave = wave_index(), waves = blockDim.x / kWave;
    const Place at = place_of(p, words, lane, lds);
    const int64_t n0 = (at.chunk * waves + wave) * kSteps;
    Part<T, kReset, 3> part;
    part.load(p, at, n0, lane, nullptr, 0, 0, nullptr, p.initial);
    const Published of(p, at, words, lane);
    Early early;
    early.load(of, wave, waves);
    __builtin_amdgcn_sched_barrier(0);  // every load is on its way before the first wait

    const int left = part.left;
    const float k = p.rates ? part.decay : open_log2(part.decay, p.rate);
    float a[kSteps], in[kSteps];
    Pair own{1.0f, 0.0f};
    for_part(left, [&](auto full) {
#pragma unroll
        for (int s = 0; s < kSteps; ++s) {
            const bool there = full.value || s < left, drop = kReset && (part.resets >> s & 1);
            const Gates g = gates(static_cast<float>(part.e[0][s]), static_cast<float>(part.e[1][s]), k);
            a[s] = there ? g.a : 1.0f;
            in[s] = there ? g.s * g.open_i * static_cast<float>(part.e[2][s]) : 0.0f;
            own.a = drop ? -0.0f : own.a * a[s];
            own.b = drop ? in[s] : fmaf(a[s], own.b, in[s]);
        }
    });
    lds.parts[wave][lane] = own;
    __syncthreads();
    float h = join_chunks<false, kReset>(p, at, of, early, lane, wave, waves, part.initial, lds);
    for (int w = 0; w < wave; ++w) h = lds.parts[w][lane].after<kReset>(h);
    if (left > 0) {
        const float *out = starts + (at.b * cdiv(p.time, kSteps) + n0 / kSteps) * p.channels + at.c0;
        store_channel<float>(buffer_of(out, starts), at.channel, 0, h);
        Rows to = rows_of<T>(p, at, n0, left, y, p.time * p.channels, p.channels);
#pragma unroll
        for (int s = 0; s < kSteps; ++s) {
            const bool drop = kReset && (part.resets >> s & 1);
            h = drop ? in[s] : fmaf(a[s], h, in[s]);
            // (a step past the end leaves h and writes the last row again)
            store_channel<T>(to.buffer, at.channel, to.next(), h);
        }
    }
    if (last && wave == waves - 1 && at.chunk == p.chunks - 1) {
        store_channel<float>(buffer_of(last + at.b * p.channels + at.c0, true), at.channel, 0, h);
    }
}

// 16 x 3751 x 960 bfloat16: 216 us (median; 201 to 234 by run and card), 3.8 TB/s,
// where the same moves alone took 173 and the vector units issue for 136.
//
// G as a carry c between steps: g = dy + c, c = a g (0 at a reset), from the
// last step to the first; chunk 0 of the fold is the last in time.
template <class T, bool kReset>
__global__ void __launch_bounds__(kMaxWaves *kWave)
    recurrence_bwd_kernel(RecArgs p, const T *gy, int64_t sgb, int64_t sgt, const float *g_last,
                          const float *starts, T *gx, T *gr, T *gi, float *decay_part,
                          float *g_initial, uint64_t *words) {
    __shared__ Shared lds;
    __shared__ float sums[kMaxWaves][kWave];
    const int lane = lane_id(), wave = wave_index(), waves = blockDim.x / kWave;
    const Place at = place_of(p, words, lane, lds);
    const int64_t n0 = ((p.chunks - 1 - at.chunk) * waves + wave) * kSteps;
    Part<T, kReset, 4> part;
    part.load(p, at, n0, lane, gy, sgb, sgt, starts, g_last);
    const Published of(p, at, words, lane);
    Early early;
    early.load(of, wave, waves);
    __builtin_amdgcn_sched_barrier(0);  // every load is on its way before the first wait

    const int left = part.left;
    const float k = p.rates ? part.decay : open_log2(part.decay, p.rate);
    float open_r[kSteps], a[kSteps], g[kSteps];
    Pair own{1.0f, 0.0f};
    for_part(left, [&](auto full) {
#pragma unroll
        for (int s = kSteps - 1; s >= 0; --s) {
            const bool there = full.value || s < left, drop = kReset && (part.resets >> s & 1);
            open_r[s] = sigmoid_fast(static_cast<float>(part.e[0][s]));
            a[s] = exp2_fast(k * open_r[s]);
            g[s] = there ? static_cast<float>(part.e[3][s]) : 0.0f;
            const float on = there ? a[s] : 1.0f;
            own.a = drop ? -0.0f : own.a * on;
            own.b = drop ? 0.0f : on * (g[s] + own.b);
        }
    });
    lds.parts[wave][lane] = own;
    __syncthreads();
    float c = join_chunks<true, kReset>(p, at, of, early, lane, wave, waves, part.initial, lds), sum = 0.0f;
    for (int w = waves - 1; w > wave; --w) c = lds.parts[w][lane].after<kReset>(c);
    for_part(left, [&](auto full) {
#pragma unroll
        for (int s = kSteps - 1; s >= 0; --s) {
            const bool there = full.value || s < left, drop = kReset && (part.resets >> s & 1);
            g[s] += c;
            c = drop ? 0.0f : there ? a[s] * g[s] : c;
        }
        const int64_t sb = p.time * p.channels;
        Rows to_x = rows_of<T>(p, at, n0, left, gx, sb, p.channels);
        Rows to_i = rows_of<T>(p, at, n0, left, gi, sb, p.channels);
        Rows to_r = rows_of<T>(p, at, n0, left, gr, sb, p.channels);
        float h = part.start;
#pragma unroll
        for (int s = 0; s < kSteps; ++s) {
            if (!full.value && s >= left) continue;
            const float x = static_cast<float>(part.e[2][s]);
            const float open_i = sigmoid_fast(static_cast<float>(part.e[1][s]));
            const float log2a = k * open_r[s];
            const float scale = input_scale(log2a, a[s]);
            const float before = kReset && (part.resets >> s & 1) ? 0.0f : h;
            const float gate = scale * open_i, kept = a[s] * before;
            const float driven = g[s] * gate * x;
            // a^2 / s^2 is infinite where u is 0; times s u (1 - open) it tends to 0
            const float slope = scale > 0.0f ? a[s] * a[s] * rcp_fast(scale * scale) : 0.0f;
            const float du = fmaf(slope, driven, -kept * g[s]);
            sum = fmaf(du, open_r[s], sum);
            h = fmaf(gate, x, kept);
            store_channel<T>(to_x.buffer, at.channel, to_x.next(), g[s] * gate);
            store_channel<T>(to_i.buffer, at.channel, to_i.next(), fmaf(-driven, open_i, driven));
            store_channel<T>(to_r.buffer, at.channel, to_r.next(), du * (-kLn2 * log2a) * (1.0f - open_r[s]));
        }
    });
    if (g_initial && wave == 0 && at.chunk == p.chunks - 1) {
        store_channel<float>(buffer_of(g_initial + at.b * p.channels + at.c0, true), at.channel, 0, c);
    }
    // the chunk's share of ddecay
    sums[wave][lane] = sum;
    __syncthreads();
    if (wave == 0) {
        for (int w = 1; w < waves; ++w) sum += sums[w][lane];
        float *out = decay_part + (at.chunk * p.batch + at.b) * p.channels + at.c0;
        store_channel<float>(buffer_of(out, true), at.channel, 0, sum);
    }
}

// ddecay from the chunks' shares
__global__ void __launch_bounds__(kSumShares *kSumColumns)
    recurrence_decay_kernel(const float *part, int64_t rows, int64_t channels, const float *decay,
                            float rate, float *g_decay) {
    const int64_t c = int64_t(blockIdx.x) * kSumColumns + threadIdx.x % kSumColumns;
    const float sum = sum_parts(part, rows, channels, c, channels);
    // (the exact sigmoid: its error would be the whole sum's)
    if (threadIdx.x < kSumColumns && c < channels) g_decay[c] = sum * (rate / (1.0f + expf(-decay[c])));
}

// kPending into all words, and open_log2 of every channel into rates
__global__ void __launch_bounds__(256)
    recurrence_fill_kernel(uint64_t *words, int64_t count, const float *decay, int64_t channels, float rate,
                           float *rates) {
    const int64_t first = int64_t(blockIdx.x) * 256 + threadIdx.x, step = int64_t(gridDim.x) * 256;
    for (int64_t c = first; c < channels; c += step) rates[c] = open_log2(decay[c], rate);
    for (int64_t k = first; k < count; k += step) words[k] = kPending;
}

template <class T>
__global__ void __launch_bounds__(kRecThreads) recurrence_step_kernel(RecArgs p, float *state, T *y) {
    const int64_t c = int64_t(blockIdx.x) * kRecThreads + threadIdx.x, b = blockIdx.y;
    if (c >= p.channels) return;
    const Gates g = gates(*at<T>(p.r, b, p.srb, 0, 0, c), *at<T>(p.i, b, p.sib, 0, 0, c),
                          open_log2(p.decay[c], p.rate));
    const float x = *at<T>(p.x, b, p.sxb, 0, 0, c);
    const float h = fmaf(g.a, state[b * p.channels + c], g.s * g.open_i * x);
    state[b * p.channels + c] = h;
    y[b * p.channels + c] = static_cast<T>(h);
}

// ---------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------

// in bytes, so that the offset of a part's last row stays below 2^31
constexpr int64_t kMostStride = int64_t(1) << 27;
static_assert((kSteps - 1) * kMostStride <= kBufferBytes);

static bool near_steps(int64_t stride, int dtype) { return stride < kMostStride / type_size(dtype); }

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
    PESQ_CHECK_ARG(p->rate > 0.0 && p->rate <= 0x1p126,  // (float32, times log2(e))
                   "the rate has to be positive and at most 2^126, got %g", p->rate);
    for (int k = 0; k < 6; ++k) {
        PESQ_CHECK_ARG(p->strides[k / 2][k % 2] >= 0, "negative stride");
        PESQ_CHECK_ARG(k % 2 == 0 || near_steps(p->strides[k / 2][1], p->dtype),
                       "steps are less than 2^27 bytes apart, got %lld elements", (long long)p->strides[k / 2][1]);
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

// How a call is cut up; waves: of a workgroup.
struct Plan {
    int waves;
    int64_t chunks, groups;
    int64_t words, bytes;  // of the pairs; of the scratch: these and the channels' rates
};

static Plan plan_of(const pesq_recurrence *p) {
    Plan plan;
    plan.groups = cdiv(p->channels, kWave);
    const int64_t parts = cdiv(p->time, kSteps);
    // Few wavefronts leave room for several workgroups on a compute unit, of which
    // some compute while others wait (16 x 3751 x 960 bfloat16, forward and backward:
    // 356 us with 4, 380 us with 8); many keep the chunks of a long row, and the pairs
    // to fold, few.  Forward and backward in bfloat16, with 16 / with 4:
    //   1 x 64000 x 65    75 /  98 us      2 x 120000 x 256   448 / 579 us
    //   1 x 64000 x 512  242 / 275 us      4 x 32000 x 512    453 / 465 us
    //   8 x 20000 x 1024  1055 / 1033 us   16 x 17000 x 512   905 / 876 us
    // so the length decides, and rows just past kLongRow in large batches lose 2 to 3 %.
    const int most = parts / kWaves > kLongRow ? kMaxWaves : kWaves;
    plan.waves = parts < most ? static_cast<int>(parts < 1 ? 1 : parts) : most;
    plan.chunks = parts < 1 ? 1 : cdiv(parts, plan.waves);
    plan.words = plan.chunks == 1 ? 0
                                  : kCounters * kCounterStride +
                                        (plan.chunks + plan.chunks / kFan) * p->batch * plan.groups * kWave;
    plan.bytes = plan.words == 0 ? 0 : (plan.words + cdiv(p->channels, 2)) * int64_t(sizeof(uint64_t));
    return plan;
}

static RecArgs kernel_args(const pesq_recurrence *p, const Plan &plan) {
    return {p->batch, p->time, p->channels, p->x, p->recur_gate, p->input_gate,
            p->strides[0][0], p->strides[0][1], p->strides[1][0], p->strides[1][1],
            p->strides[2][0], p->strides[2][1], p->decay, p->initial, p->reset,
            static_cast<float>(p->rate), p->reverse != 0, plan.chunks,
            static_cast<int32_t>(plan.groups), nullptr};
}

static int check_grid(const pesq_recurrence *p, const Plan &plan) {
    PESQ_CHECK_ARG(plan.chunks * p->batch * plan.groups * plan.waves * kWave < (int64_t(1) << 32),
                   "a recurrence of %lld x %lld x %lld is too large", (long long)p->batch,
                   (long long)p->time, (long long)p->channels);
    return PESQ_OK;
}

// fn(T(), reset) with reset as a constant
template <class Fn>
static void with_variant(const pesq_recurrence *p, Fn fn) {
    with_type(p->dtype, [&](auto type) {
        if (p->reset) {
            fn(type, std::true_type());
        } else {
            fn(type, std::false_type());
        }
    });
}

// Makes the scratch of a call of several chunks a row ready, and the rates known to it
static void fill_words(RecArgs &args, const Plan &plan, uint64_t *words, hipStream_t stream) {
    if (plan.words == 0) return;
    float *rates = reinterpret_cast<float *>(words + plan.words);
    const int64_t blocks = cdiv(plan.words, 1024);
    recurrence_fill_kernel<<<static_cast<unsigned>(blocks < 2048 ? blocks : 2048), 256, 0, stream>>>(
        words, plan.words, args.decay, args.channels, args.rate, rates);
    args.rates = rates;
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
    const Plan plan = plan_of(p);
    if (starts) *starts = states * cdiv(p->time, kSteps);
    if (forward) *forward = plan.bytes;
    if (backward) *backward = plan.bytes + states * plan.chunks;
    return PESQ_OK;
}

extern "C" int pesq_recurrence_forward(const pesq_recurrence *p, void *y, float *last,
                                       float *starts, void *workspace, hipStream_t stream) {
    if (int st = check_operands(p)) return st;
    if (empty(p)) return PESQ_OK;
    PESQ_CHECK_ARG(y || p->time == 0, "null argument");
    const Plan plan = plan_of(p);
    if (int st = check_grid(p, plan)) return st;
    PESQ_CHECK_ARG(workspace || plan.words == 0, "null argument");
    uint64_t *words = static_cast<uint64_t *>(workspace);
    RecArgs args = kernel_args(p, plan);
    fill_words(args, plan, words, stream);
    with_variant(p, [&](auto type, auto reset) {
        using T = decltype(type);
        recurrence_fwd_kernel<T, reset.value>
            <<<grid_of(p, plan), plan.waves * kWave, 0, stream>>>(
                args, static_cast<T *>(y), last, starts, words);
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
    PESQ_CHECK_ARG(!g_y || (g_strides && g_strides[0] >= 0 && g_strides[1] >= 0 &&
                            near_steps(g_strides[1], p->dtype)),
                   "the upstream gradient needs its strides");
    if (p->channels == 0) return PESQ_OK;
    PESQ_CHECK_ARG(empty(p) || (workspace && (starts || p->time == 0)), "null argument");
    PESQ_CHECK_ARG(!g_decay || p->decay, "null argument");
    const Plan plan = plan_of(p);
    if (int st = check_grid(p, plan)) return st;
    uint64_t *words = static_cast<uint64_t *>(workspace);
    float *part = reinterpret_cast<float *>(static_cast<char *>(workspace) + plan.bytes);
    if (p->batch > 0) {
        RecArgs args = kernel_args(p, plan);
        fill_words(args, plan, words, stream);
        with_variant(p, [&](auto type, auto reset) {
            using T = decltype(type);
            recurrence_bwd_kernel<T, reset.value>
                <<<grid_of(p, plan), plan.waves * kWave, 0, stream>>>(
                    args, static_cast<const T *>(g_y), g_y ? g_strides[0] : 0,
                    g_y ? g_strides[1] : 0, g_last, starts, static_cast<T *>(g_x),
                    static_cast<T *>(g_recur), static_cast<T *>(g_input), part, g_initial, words);
        });
        PESQ_CHECK_LAUNCH("pesq_recurrence_backward");
    }
    if (g_decay) {
        recurrence_decay_kernel<<<static_cast<unsigned>(cdiv(p->channels, kSumColumns)),
                                  kSumShares * kSumColumns, 0, stream>>>(
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
