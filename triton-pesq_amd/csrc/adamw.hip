// One AdamW step over many tensors, moments in 32 or in 8 bits.
//
//   m = b1 m + (1 - b1) g          v = b2 v + (1 - b2) g^2
//   p = (1 - lr wd) p - lr / (1 - b1^t) m / (sqrt(v / (1 - b2^t)) + eps)
//
// in float32, each product and sum rounded as written (no fused steps), so that
// the moments are those of the same formula in plain float32 operations.
// Elementwise and bound by memory (47.7 M bfloat16 weights with 8 bit moments:
// 96 to 105 us by card, 4.5 to 5.0 TB/s, the rate of a large copy).
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

// what of a step's factors depends on its number
struct Corrections {
    float step_size, root;
};

struct AdamArgs {
    float b1, c1, b2, c2, keep, eps;
    Corrections of_step;
};

__host__ __device__ inline Corrections corrections_of(double lr, double beta1, double beta2, double step) {
    return {static_cast<float>(lr / (1.0 - pow(beta1, step))),
            static_cast<float>(1.0 / sqrt(1.0 - pow(beta2, step)))};
}

// A launch takes up to kTensors tensors as kernel arguments: no table to copy to
// the GPU, and new gradients each step cost nothing.  Workgroups go by tiles of
// kAdamThreads lanes; a tile's tensor is found by bisection.
constexpr int kTensors = 96;
constexpr int kAdamThreads = 256;

// Neighbours that a lane takes.  With 8 bit moments 8, a block to each half of a
// wavefront: fewer and wider moves, and the scales' maxima and reciprocals shared
// by more (47.7 M bfloat16 parameters 96 us; with 4 121 us, with 16, and half the
// wavefronts at a time, 105 us).  With float32 moments 4, a move of 16 bytes that
// continues its neighbour lane's (26 tensors, 1.4 M parameters, 9.1 us; with 8
// 10.3 us), as in the kernel that writes the moments' values (76 us; 85 us).
constexpr int lane_elements(bool eight) { return eight ? 8 : 4; }
constexpr int tile_elements(bool eight) { return lane_elements(eight) * kAdamThreads; }
constexpr int kHalfLane = kBlock / (kWave / 2);
static_assert(lane_elements(true) == kHalfLane, "block_scale joins the halves of wavefronts");

struct AdamTensor {
    void *param;
    const void *grad;
    int64_t count;
    uint32_t block;  // its first one in the moments
    uint32_t end;    // number of the tile after its last one
};

struct AdamList {
    AdamTensor tensors[kTensors];
    int count;
    void *m, *v;
    float *m_scale, *v_scale;
    AdamArgs args;
    const Corrections *corrections;  // of each tensor where the GPU counts the steps, or NULL
};
static_assert(sizeof(AdamList) <= 4096, "kernel arguments");

// as written: no contraction into fused multiply-adds
#pragma clang fp contract(off)

__device__ __forceinline__ float adamw(float p, float g, float &m, float &v, const AdamArgs &a,
                                       const Corrections &c) {
    m = m * a.b1 + g * a.c1;
    v = v * a.b2 + (g * g) * a.c2;
    // The hardware's root and reciprocal, each within one unit in the last place.
    // A second moment below 2^-120, where float32 soon has fewer digits and the
    // root flushes them, counts as 2^-120: with eps = 0 there is still a quotient.
    // (a NaN, as all of a block are whose scale is infinite, stays one)
    const float held = v < 0x1p-120f ? 0x1p-120f : v;
    const float update = m * rcp_fast(__builtin_amdgcn_sqrtf(held) * c.root + a.eps);
    return p * a.keep - update * c.step_size;
}

// a lane's codes, and its moments in float32
template <int E>
struct alignas(E) Codes {
    uint32_t v[E / 4];
};
template <int E>
struct alignas(16) Lane {
    float v[E];
};

// what the codes stand for
template <int E>
__device__ __forceinline__ void values(const Codes<E> &cm, const Codes<E> &cv, float sm, float sv, Lane<E> &m,
                                       Lane<E> &v) {
#pragma unroll
    for (int k = 0; k < E; ++k) {
        const float part =
            (static_cast<float>((cm.v[k / 4] ^ 0x80808080u) >> 8 * (k % 4) & 0xff) - 128.0f) * (1.0f / 127.0f);
        m.v[k] = fabsf(part) * part * sm;
        float root = static_cast<float>(cv.v[k / 4] >> 8 * (k % 4) & 0xff) * (1.0f / 255.0f);
        root = root * root;
        v.v[k] = root * root * sv;
    }
}

// Codes are those of correctly rounded roots.  The hardware's root (one unit in
// the last place) gives the same code unless the product lies next to the middle
// between two: within 127 2^-22 of it for the first moment and 255 2^-22 for the
// second's two roots, twice the errors that can arise.  A wavefront with such an
// element, one in ten, does its codes again.

// the middle between two codes, seen from a number of codes
__device__ __forceinline__ bool near_middle(float q, float distance) {
    return fabsf(__builtin_amdgcn_fractf(q) - 0.5f) <= distance;
}

// Bytes of a lane's elements: int8 and uint8 codes.  A number of codes is
// rounded to the nearest one and clamped by the conversion that packs it; the
// first moment's are 128 up while they are packed.
template <bool kExact, int E>
__device__ __forceinline__ bool codes(const Lane<E> &m, const Lane<E> &v, float im, float iv, Codes<E> &cm,
                                      Codes<E> &cv) {
    bool near = false;
    const float least = iv == 0.0f ? 0.0f : 1.0f;
#pragma unroll
    for (int k = 0; k < E; ++k) {
        uint32_t &word_m = cm.v[k / 4], &word_v = cv.v[k / 4];
        if (k % 4 == 0) word_m = word_v = 0;
        const float ym = fabsf(m.v[k]) * im, yv = v.v[k] * iv;
        float qm, qv;
        if (kExact) {
            qm = 128.0f + copysignf(rintf(sqrtf(ym) * 127.0f), m.v[k]);
            qv = rintf(sqrtf(sqrtf(yv)) * 255.0f);
        } else {
            qm = fmaf(copysignf(__builtin_amdgcn_sqrtf(ym), m.v[k]), 127.0f, 128.0f);
            qv = __builtin_amdgcn_sqrtf(__builtin_amdgcn_sqrtf(yv)) * 255.0f;
            const bool near_m = near_middle(qm, 127.0f * 0x1p-22f), near_v = near_middle(qv, 255.0f * 0x1p-22f);
            near = near | near_m | near_v;  // (no branch between elements)
        }
        qv = fmaxf(qv, v.v[k] > 0.0f ? least : 0.0f);
        word_m = __builtin_amdgcn_cvt_pk_u8_f32(qm, k % 4, word_m);
        word_v = __builtin_amdgcn_cvt_pk_u8_f32(qv, k % 4, word_v);
        if (k % 4 == 3) word_m ^= 0x80808080u;
    }
    return near;
}

template <int kCtrl>
__device__ __forceinline__ uint32_t max_ror(uint32_t v) {
    const uint32_t other = static_cast<uint32_t>(
        __builtin_amdgcn_update_dpp(0, static_cast<int>(v), kCtrl, 0xF, 0xF, true));
    return other > v ? other : v;
}

// largest magnitude of the block in a half of a wavefront, NaN above all (its bits
// are the largest); 0 where it is too small to be held
__device__ __forceinline__ float block_scale(const Lane<kHalfLane> &f) {
    uint32_t bits = 0;
#pragma unroll
    for (int k = 0; k < kHalfLane; ++k) {
        const uint32_t other = __float_as_uint(f.v[k]) & 0x7fffffffu;
        bits = other > bits ? other : bits;
    }
    bits = max_ror<0x128>(bits);  // row_ror:8, 4, 2, 1
    bits = max_ror<0x124>(bits);
    bits = max_ror<0x122>(bits);
    bits = max_ror<0x121>(bits);
    const auto rows = __builtin_amdgcn_permlane16_swap(bits, bits, false, false);  // of the half
    bits = rows[0] > rows[1] ? rows[0] : rows[1];
    const float scale = __uint_as_float(bits);
    return scale < kSmallest ? 0.0f : scale;
}

__device__ __forceinline__ float inverse_of(float scale) { return scale == 0.0f ? 0.0f : 1.0f / scale; }

// a lane's neighbours from element `at` of a tensor; zeros past its end
template <int E, class T>
__device__ __forceinline__ void load_lane(const T *p, int64_t at, int64_t count, Lane<E> &out) {
    if (at + E <= count) {
        const auto e = load_neighbours<T, E>(p + at);
#pragma unroll
        for (int k = 0; k < E; ++k) out.v[k] = static_cast<float>(e.v[k]);
    } else {
#pragma unroll
        for (int k = 0; k < E; ++k) out.v[k] = at + k < count ? static_cast<float>(p[at + k]) : 0.0f;
    }
}

template <int E, class T>
__device__ __forceinline__ void store_lane(T *p, int64_t at, int64_t count, const Lane<E> &f) {
    if (at + E <= count) {
        Neighbours<T, E> e;
#pragma unroll
        for (int k = 0; k < E; ++k) e.v[k] = static_cast<T>(f.v[k]);
        store_neighbours<T, E>(p + at, e);
    } else {
#pragma unroll
        for (int k = 0; k < E; ++k) {
            if (at + k < count) p[at + k] = static_cast<T>(f.v[k]);
        }
    }
}

// The moments' arrays have whole blocks, whose elements past a tensor's end are
// and stay 0.
template <class T, bool kEight>
__global__ void __launch_bounds__(kAdamThreads) adamw_kernel(AdamList list) {
    constexpr int E = lane_elements(kEight), kRow = kBlock / E;  // kRow lanes to a block
    int low = 0, high = list.count - 1;
    while (low < high) {
        const int middle = (low + high) / 2;
        if (blockIdx.x < list.tensors[middle].end) {
            high = middle;
        } else {
            low = middle + 1;
        }
    }
    const AdamTensor &t = list.tensors[low];
    const uint32_t tile = blockIdx.x - (low ? list.tensors[low - 1].end : 0);
    const int64_t at = (int64_t(tile) * kAdamThreads + threadIdx.x) * E, count = t.count;
    if (at / kBlock * kBlock >= count) return;  // (all lanes of a block)
    T *param = static_cast<T *>(t.param);
    const T *grad = static_cast<const T *>(t.grad);
    const AdamArgs a = list.args;
    const Corrections c = list.corrections ? list.corrections[low] : a.of_step;
    const int64_t held = t.block + at / kBlock, mine = int64_t(t.block) * kRow + at / E;
    Lane<E> p, g, m, v;
    load_lane(param, at, count, p);
    load_lane(grad, at, count, g);
    if constexpr (kEight) {
        values(static_cast<const Codes<E> *>(list.m)[mine], static_cast<const Codes<E> *>(list.v)[mine],
               list.m_scale[held], list.v_scale[held], m, v);
    } else {
        m = static_cast<const Lane<E> *>(list.m)[mine];
        v = static_cast<const Lane<E> *>(list.v)[mine];
    }
    // (past the end m, v and g are 0, and the moments stay 0)
#pragma unroll
    for (int k = 0; k < E; ++k) p.v[k] = adamw(p.v[k], g.v[k], m.v[k], v.v[k], a, c);
    store_lane(param, at, count, p);
    if constexpr (kEight) {
        const float sm = block_scale(m), sv = block_scale(v);
        const float im = inverse_of(sm), iv = inverse_of(sv);
        Codes<E> cm, cv;
        if (__any(codes<false>(m, v, im, iv, cm, cv))) codes<true>(m, v, im, iv, cm, cv);
        static_cast<Codes<E> *>(list.m)[mine] = cm;
        static_cast<Codes<E> *>(list.v)[mine] = cv;
        if (at % kBlock == 0) {
            list.m_scale[held] = sm;
            list.v_scale[held] = sv;
        }
    } else {
        static_cast<Lane<E> *>(list.m)[mine] = m;
        static_cast<Lane<E> *>(list.v)[mine] = v;
    }
}

// Counts of a launch's tensors that the GPU keeps, each up by one, and what follows
// from them: a captured step's replays are steps of their own.
struct CountList {
    int64_t *steps[kTensors];
    int count;
    double lr, beta1, beta2;
};

__global__ void __launch_bounds__(kTensors) adamw_count_kernel(CountList list, Corrections *corrections) {
    const int k = threadIdx.x;
    if (k >= list.count) return;
    // (past the GPU's caches: the host writes there between launches)
    const int64_t step = __hip_atomic_load(list.steps[k], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_SYSTEM) + 1;
    __hip_atomic_store(list.steps[k], step, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_SYSTEM);
    corrections[k] = corrections_of(list.lr, list.beta1, list.beta2, static_cast<double>(step));
}

constexpr int kValues = 4;  // of a lane
__global__ void __launch_bounds__(kAdamThreads)
    adamw_moments_kernel(const Codes<kValues> *m, const Codes<kValues> *v, const float *m_scale,
                         const float *v_scale, int64_t blocks, Lane<kValues> *m_out, Lane<kValues> *v_out) {
    const int64_t mine = int64_t(blockIdx.x) * kAdamThreads + threadIdx.x, block = mine * kValues / kBlock;
    if (block >= blocks) return;
    Lane<kValues> em, ev;
    values(m[mine], v[mine], m_scale[block], v_scale[block], em, ev);
    m_out[mine] = em;
    v_out[mine] = ev;
}

// the launch of a list of `tiles` tiles
static void launch_adamw(const AdamList &list, int dtype, bool eight, uint32_t tiles, hipStream_t stream) {
    with_type(dtype, [&](auto type) {
        using T = decltype(type);
        if (eight) {
            adamw_kernel<T, true><<<tiles, kAdamThreads, 0, stream>>>(list);
        } else {
            adamw_kernel<T, false><<<tiles, kAdamThreads, 0, stream>>>(list);
        }
    });
}

}  // namespace pesq

using namespace pesq;

static constexpr int64_t kMostTiles = (int64_t(1) << 32) / kAdamThreads - 1;  // workgroups of a launch

// steps and corrections: of pesq_adamw_step_counted, or NULL
static int adamw_step(const pesq_adamw_tensor *tensors, int64_t count, const pesq_adamw_options *o,
                      int64_t *const *steps, Corrections *corrections, void *exp_avg, void *exp_avg_sq,
                      float *exp_avg_scale, float *exp_avg_sq_scale, hipStream_t stream) {
    PESQ_CHECK_ARG(o != nullptr && count >= 0 && (tensors || count == 0), "null argument");
    PESQ_CHECK_ARG(known_type(o->dtype), "unknown element type %d", int(o->dtype));
    PESQ_CHECK_ARG(o->state_bits == 32 || o->state_bits == 8, "moments have 32 or 8 bits, got %d",
                   int(o->state_bits));
    PESQ_CHECK_ARG(steps || o->step >= 1, "steps count from 1, got %lld", (long long)o->step);
    PESQ_CHECK_ARG(o->beta1 >= 0.0 && o->beta1 < 1.0 && o->beta2 >= 0.0 && o->beta2 < 1.0,
                   "betas have to be in [0, 1)");
    const bool eight = o->state_bits == 8;
    const int64_t tile = tile_elements(eight);
    const bool arrays = exp_avg && exp_avg_sq && (!eight || (exp_avg_scale && exp_avg_sq_scale));
    for (const void *array : {exp_avg, exp_avg_sq}) {
        PESQ_CHECK_ARG(reinterpret_cast<uintptr_t>(array) % 16 == 0, "the moments start at multiples of 16 bytes");
    }
    for (int64_t k = 0; k < count; ++k) {
        PESQ_CHECK_ARG(tensors[k].count >= 0 && tensors[k].first >= 0 && tensors[k].first % kBlock == 0,
                       "tensor %lld has no place in the moments", (long long)k);
        PESQ_CHECK_ARG(tensors[k].count == 0 || (arrays && tensors[k].param && tensors[k].grad), "null argument");
        PESQ_CHECK_ARG(tensors[k].count <= kMostTiles * tile && tensors[k].first < (int64_t(1) << 40),
                       "tensor %lld is too large", (long long)k);
    }
    const AdamArgs a{static_cast<float>(o->beta1), static_cast<float>(1.0 - o->beta1),
                     static_cast<float>(o->beta2), static_cast<float>(1.0 - o->beta2),
                     static_cast<float>(1.0 - o->lr * o->weight_decay),
                     static_cast<float>(o->eps),
                     steps ? Corrections{} : corrections_of(o->lr, o->beta1, o->beta2, static_cast<double>(o->step))};
    AdamList list;
    list.count = 0;
    list.m = exp_avg;
    list.v = exp_avg_sq;
    list.m_scale = exp_avg_scale;
    list.v_scale = exp_avg_sq_scale;
    list.args = a;
    list.corrections = corrections;
    int64_t tiles = 0;
    const auto launch = [&](int64_t end) -> int {  // of the list, whose tensors are those before `end`
        if (steps) {
            CountList counts;
            counts.count = list.count;
            counts.lr = o->lr;
            counts.beta1 = o->beta1;
            counts.beta2 = o->beta2;
            for (int k = 0; k < list.count; ++k) counts.steps[k] = steps[end - list.count + k];
            adamw_count_kernel<<<1, kTensors, 0, stream>>>(counts, corrections + (end - list.count));
            list.corrections = corrections + (end - list.count);
        }
        if (tiles > 0) launch_adamw(list, o->dtype, eight, static_cast<uint32_t>(tiles), stream);
        if (steps || tiles > 0) PESQ_CHECK_LAUNCH("pesq_adamw_step");
        list.count = 0;
        tiles = 0;
        return PESQ_OK;
    };
    for (int64_t k = 0; k < count; ++k) {
        const pesq_adamw_tensor &t = tensors[k];
        const int64_t more = cdiv(t.count, tile);
        if (list.count == kTensors || tiles + more > kMostTiles) {
            if (int st = launch(k)) return st;
        }
        // (one without elements has no tile, and is found by none)
        tiles += more;
        list.tensors[list.count++] = {t.param, t.grad, t.count, static_cast<uint32_t>(t.first / kBlock),
                                      static_cast<uint32_t>(tiles)};
    }
    return list.count > 0 ? launch(count) : PESQ_OK;
}

extern "C" int pesq_adamw_step(const pesq_adamw_tensor *tensors, int64_t count,
                               const pesq_adamw_options *o, void *exp_avg, void *exp_avg_sq,
                               float *exp_avg_scale, float *exp_avg_sq_scale, hipStream_t stream) {
    return adamw_step(tensors, count, o, nullptr, nullptr, exp_avg, exp_avg_sq, exp_avg_scale, exp_avg_sq_scale,
                      stream);
}

extern "C" int pesq_adamw_step_counted(const pesq_adamw_tensor *tensors, int64_t count,
                                       const pesq_adamw_options *o, int64_t *const *steps, float *corrections,
                                       void *exp_avg, void *exp_avg_sq, float *exp_avg_scale,
                                       float *exp_avg_sq_scale, hipStream_t stream) {
    if (count == 0) return PESQ_OK;
    PESQ_CHECK_ARG(count > 0 && steps && corrections, "null argument");
    PESQ_CHECK_ARG(reinterpret_cast<uintptr_t>(corrections) % 8 == 0, "the corrections start at a multiple of 8 bytes");
    for (int64_t k = 0; k < count; ++k) PESQ_CHECK_ARG(steps[k], "tensor %lld has no count", (long long)k);
    return adamw_step(tensors, count, o, steps, reinterpret_cast<Corrections *>(corrections), exp_avg, exp_avg_sq,
                      exp_avg_scale, exp_avg_sq_scale, stream);
}

extern "C" int pesq_adamw_moments(const void *exp_avg, const void *exp_avg_sq,
                                  const float *exp_avg_scale, const float *exp_avg_sq_scale,
                                  int64_t count, float *m, float *v, hipStream_t stream) {
    PESQ_CHECK_ARG(count >= 0 && count % kBlock == 0 && count <= kMostTiles * kAdamThreads * kValues,
                   "whole blocks of %d elements, 2^34 - 1024 elements at most, got %lld", kBlock, (long long)count);
    if (count == 0) return PESQ_OK;
    PESQ_CHECK_ARG(exp_avg && exp_avg_sq && exp_avg_scale && exp_avg_sq_scale && m && v, "null argument");
    for (const void *array : {exp_avg, exp_avg_sq, static_cast<const void *>(m), static_cast<const void *>(v)}) {
        PESQ_CHECK_ARG(reinterpret_cast<uintptr_t>(array) % 16 == 0, "the moments start at multiples of 16 bytes");
    }
    const int64_t blocks = count / kBlock;
    adamw_moments_kernel<<<static_cast<unsigned>(cdiv(count, kAdamThreads * kValues)), kAdamThreads, 0, stream>>>(
        static_cast<const Codes<kValues> *>(exp_avg), static_cast<const Codes<kValues> *>(exp_avg_sq), exp_avg_scale,
        exp_avg_sq_scale, blocks, reinterpret_cast<Lane<kValues> *>(m), reinterpret_cast<Lane<kValues> *>(v));
    PESQ_CHECK_LAUNCH("pesq_adamw_moments");
    return PESQ_OK;
}
