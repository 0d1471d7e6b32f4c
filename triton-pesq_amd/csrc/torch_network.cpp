// PyTorch autograd nodes and entry points of the operators of the networks
// that the loss trains, in C++ for the reason torch_autograd.cpp gives.
//
// Each entry point checks its tensors, allocates outputs and workspaces on the
// caller's device and enqueues the library's calls on PyTorch's current stream.

#include "torch_common.hpp"

#include <array>
#include <optional>
#include <type_traits>
#include <vector>

namespace {

using OptTensor = std::optional<at::Tensor>;

int type_code(const at::Tensor &t, const char *what) {
    switch (t.scalar_type()) {
        case at::kFloat: return PESQ_F32;
        case at::kBFloat16: return PESQ_BF16;
        case at::kHalf: return PESQ_F16;
        default: break;
    }
    TORCH_CHECK(false, what, " has to be float32, bfloat16 or float16, got ", t.scalar_type());
}

void check_gpu(const at::Tensor &t, const char *what, const at::Tensor &like) {
    TORCH_CHECK(t.is_cuda(), "The HIP backend needs `", what, "` to live on a GPU.");
    TORCH_CHECK(t.get_device() == like.get_device(), "`", what, "` has to be on the same GPU as `x`.");
}

// t itself where neighbours of the last axis lie next to each other
at::Tensor dense_rows(const at::Tensor &t) {
    return t.size(-1) <= 1 || t.stride(-1) == 1 ? t : t.contiguous();
}

// t itself where it has the type (`to` would cost a call's dispatch)
at::Tensor of_type(const at::Tensor &t, at::ScalarType type) {
    return t.scalar_type() == type ? t : t.to(type);
}

// a bit for each input that requires a gradient, asked for in this backward or not
template <size_t N>
int64_t requiring(const std::array<const at::Tensor *, N> &inputs) {
    int64_t bits = 0;
    for (size_t k = 0; k < N; ++k) {
        if (inputs[k]->defined() && inputs[k]->requires_grad()) bits |= int64_t(1) << k;
    }
    return bits;
}

// The gradients, with a derivative that raises where a double backward would need
// one: where an upstream gradient wants it, or an input of `requiring` that the
// gradient is a function of, by `depends` (of each gradient, in the same bits).
template <size_t N>
void mark_once(variable_list &grads, const variable_list &upstream, int64_t requiring,
               const std::array<int64_t, N> &depends) {
    if (!torch::autograd::GradMode::is_enabled()) return;
    bool needed = false;
    for (const at::Tensor &g : upstream) needed = needed || (g.defined() && g.requires_grad());
    for (size_t k = 0; k < N; ++k) {
        at::Tensor &g = grads[k];
        if (g.defined() && (needed || (requiring & depends[k]))) {
            g = OnceDifferentiable::apply(g.detach().requires_grad_(true));
        }
    }
}

// t was updated in place: a node that has saved it raises in its backward
void written(const at::Tensor &t) {
    if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

// Calls that need no node are spared it, and with it the node's refusal of forward
// mode derivatives, which the kernels do not have
void check_no_tangent(const at::Tensor &t) {
    TORCH_CHECK(!t.unsafeGetTensorImpl()->_fw_grad(0, t).defined(),
                "forward mode derivatives (jvp) are not implemented for this operator");
}

template <class... Tensors>
void check_no_tangents(const Tensors &...tensors) {
    const auto one = [](const auto &t) {
        if constexpr (std::is_same_v<std::decay_t<decltype(t)>, OptTensor>) {
            if (t) check_no_tangent(*t);
        } else {
            check_no_tangent(t);
        }
    };
    (one(tensors), ...);
}

void *data(const at::Tensor &t) { return t.defined() ? t.data_ptr() : nullptr; }

// ---------------------------------------------------------------------------
// gated linear recurrence
// ---------------------------------------------------------------------------

// x, the gates (dense rows), decay, initial and reset (undefined: none)
struct RecurrenceInputs {
    at::Tensor x, recur, input, decay, initial, reset;

    pesq_recurrence call(bool reverse, double rate) const {
        pesq_recurrence p{};
        const bool step = x.dim() == 2;
        p.batch = x.size(0);
        p.time = step ? 1 : x.size(1);
        p.channels = x.size(-1);
        p.dtype = type_code(x, "`x`");
        p.reverse = reverse;
        p.rate = rate;
        const std::array<const at::Tensor *, 3> operands{&x, &recur, &input};
        for (int k = 0; k < 3; ++k) {
            p.strides[k][0] = operands[k]->stride(0);
            p.strides[k][1] = step ? 0 : operands[k]->stride(1);
        }
        p.x = x.data_ptr();
        p.recur_gate = recur.data_ptr();
        p.input_gate = input.data_ptr();
        p.decay = decay.data_ptr<float>();
        p.initial = data_or_null<float>(initial);
        p.reset = static_cast<const uint8_t *>(data(reset));
        return p;
    }
};

void check_recurrence_inputs(const at::Tensor &x, const at::Tensor &recur, const at::Tensor &input,
                             const at::Tensor &decay, int64_t dims, const char *axes) {
    TORCH_CHECK(x.is_cuda(), "The HIP backend needs `x` to live on a GPU.");
    TORCH_CHECK(x.dim() == dims, "the gated recurrence expects x as ", axes, ", got ", x.sizes());
    type_code(x, "`x`");
    const std::array<std::pair<const char *, const at::Tensor *>, 2> gates{
        {{"recur_gate", &recur}, {"input_gate", &input}}};
    for (const auto &[name, t] : gates) {
        check_gpu(*t, name, x);
        TORCH_CHECK(t->sizes() == x.sizes(), "`", name, "` has to have the shape of x, ", x.sizes(),
                    ", got ", t->sizes());
        TORCH_CHECK(t->scalar_type() == x.scalar_type(), "`", name, "` has to have the type of x, ",
                    x.scalar_type(), ", got ", t->scalar_type());
    }
    check_gpu(decay, "decay", x);
    TORCH_CHECK(decay.is_floating_point() && decay.dim() == 1 && decay.size(0) == x.size(-1),
                "`decay` has to be a floating [channels] tensor, got ", decay.scalar_type(), " ", decay.sizes());
}

void check_state(const at::Tensor &state, const char *name, const at::Tensor &x) {
    check_gpu(state, name, x);
    TORCH_CHECK(state.scalar_type() == at::kFloat && state.dim() == 2 &&
                    state.size(0) == x.size(0) && state.size(1) == x.size(-1),
                "`", name, "` has to be float32 [batch, channels], got ", state.scalar_type(), " ",
                state.sizes());
}

// rows of neighbours, steps as near to each other as the library takes them
at::Tensor recurrence_rows(const at::Tensor &t) {
    return t.stride(1) < (int64_t(1) << 27) / t.element_size() ? dense_rows(t) : t.contiguous();
}

struct RecurrenceResult {
    RecurrenceInputs in;
    at::Tensor y, last, starts;
};

// keep: with the states that the backward reads
RecurrenceResult run_recurrence(const at::Tensor &x, const at::Tensor &recur, const at::Tensor &input,
                                const at::Tensor &decay, const OptTensor &initial,
                                const OptTensor &reset, bool reverse, double rate, bool keep) {
    const c10::DeviceGuard guard(x.device());
    RecurrenceResult r;
    r.in = {recurrence_rows(x), recurrence_rows(recur), recurrence_rows(input), decay.contiguous(),
            initial ? initial->contiguous() : at::Tensor(), reset ? reset->contiguous() : at::Tensor()};
    const pesq_recurrence p = r.in.call(reverse, rate);
    size_t starts_bytes = 0, ws_bytes = 0;
    check(pesq_recurrence_workspace(&p, &starts_bytes, &ws_bytes, nullptr),
          "pesq_recurrence_workspace");
    const auto bytes = x.options().dtype(at::kByte).requires_grad(false);
    at::Tensor ws;
    if (keep) r.starts = at::empty({static_cast<int64_t>(starts_bytes)}, bytes);
    if (ws_bytes > 0) ws = at::empty({static_cast<int64_t>(ws_bytes)}, bytes);
    r.y = at::empty(x.sizes(), x.options());
    r.last = at::empty({x.size(0), x.size(2)}, x.options().dtype(at::kFloat));
    check(pesq_recurrence_forward(&p, r.y.data_ptr(), r.last.data_ptr<float>(),
                                  static_cast<float *>(data(r.starts)), data(ws), current_stream(x)),
          "pesq_recurrence_forward");
    return r;
}

struct Recurrence : public torch::autograd::Function<Recurrence> {
    static variable_list forward(AutogradContext *ctx, const at::Tensor &x, const at::Tensor &recur,
                                 const at::Tensor &input, const at::Tensor &decay,
                                 const OptTensor &initial, const OptTensor &reset, bool reverse,
                                 double rate) {
        const RecurrenceResult r = run_recurrence(x, recur, input, decay, initial, reset, reverse, rate, true);
        ctx->set_materialize_grads(false);
        ctx->save_for_backward({r.in.x, r.in.recur, r.in.input, r.in.decay, r.in.initial, r.in.reset, r.starts});
        ctx->saved_data["reverse"] = reverse;
        ctx->saved_data["rate"] = rate;
        const at::Tensor none;
        ctx->saved_data["requiring"] = requiring<5>({&x, &recur, &input, &decay, initial ? &*initial : &none});
        return {r.y, r.last};
    }

    static variable_list backward(AutogradContext *ctx, variable_list grads) {
        variable_list out(8);  // one per argument of forward
        if (!grads[0].defined() && !grads[1].defined()) return out;
        const variable_list saved = ctx->get_saved_variables();
        const RecurrenceInputs in{saved[0], saved[1], saved[2], saved[3], saved[4], saved[5]};
        const at::Tensor &x = in.x;
        const c10::DeviceGuard guard(x.device());
        const pesq_recurrence p = in.call(ctx->saved_data["reverse"].toBool(),
                                          ctx->saved_data["rate"].toDouble());
        size_t ws_bytes = 0;
        check(pesq_recurrence_workspace(&p, nullptr, nullptr, &ws_bytes), "pesq_recurrence_workspace");
        at::Tensor ws = at::empty({static_cast<int64_t>(ws_bytes)}, x.options().dtype(at::kByte));
        at::Tensor g_y, g_last;
        {
            const at::NoGradGuard no_grad;
            if (grads[0].defined()) g_y = recurrence_rows(of_type(grads[0], x.scalar_type()));
            if (grads[1].defined()) g_last = of_type(grads[1], at::kFloat).contiguous();
        }
        for (int k = 0; k < 3; ++k) {
            if (ctx->needs_input_grad(k)) out[k] = at::empty(x.sizes(), x.options());
        }
        const auto f32 = x.options().dtype(at::kFloat);
        if (ctx->needs_input_grad(3)) out[3] = at::empty({x.size(2)}, f32);
        if (in.initial.defined() && ctx->needs_input_grad(4)) out[4] = at::empty({x.size(0), x.size(2)}, f32);
        const std::array<int64_t, 2> strides{g_y.defined() ? g_y.stride(0) : 0,
                                             g_y.defined() ? g_y.stride(1) : 0};
        check(pesq_recurrence_backward(&p, data(g_y), strides.data(), data_or_null<float>(g_last),
                                       static_cast<const float *>(data(saved[6])), data(out[0]),
                                       data(out[1]), data(out[2]), data_or_null<float>(out[3]),
                                       data_or_null<float>(out[4]), data(ws), current_stream(x)),
              "pesq_recurrence_backward");
        // G is a function of the factors a, so of the recurrence's gate and the decay;
        // x and the initial state, in which y is linear, are in the gates' alone
        constexpr int64_t kX = 1, kRecur = 2, kInput = 4, kDecay = 8, kInitial = 16;
        constexpr int64_t kFactors = kRecur | kDecay, kAll = kX | kInput | kInitial | kFactors;
        mark_once<5>(out, grads, ctx->saved_data["requiring"].toInt(),
                     {kFactors | kInput, kAll, kFactors | kInput | kX, kAll, kFactors});
        return out;
    }
};

std::vector<at::Tensor> gated_recurrence(const at::Tensor &x, const at::Tensor &recur,
                                         const at::Tensor &input, const at::Tensor &any_decay,
                                         const OptTensor &initial, const OptTensor &reset,
                                         bool reverse, double rate) {
    check_recurrence_inputs(x, recur, input, any_decay, 3, "[batch, time, channels]");
    const at::Tensor decay = of_type(any_decay, at::kFloat);
    if (initial) check_state(*initial, "initial_state", x);
    if (reset) {
        check_gpu(*reset, "reset", x);
        TORCH_CHECK(reset->scalar_type() == at::kBool && reset->dim() == 2 &&
                        reset->size(0) == x.size(0) && reset->size(1) == x.size(1),
                    "`reset` has to be bool [batch, time], got ", reset->scalar_type(), " ",
                    reset->sizes());
    }
    const bool keep = torch::autograd::GradMode::is_enabled() &&
                      (x.requires_grad() || recur.requires_grad() || input.requires_grad() ||
                       decay.requires_grad() || (initial && initial->requires_grad()));
    if (keep) return Recurrence::apply(x, recur, input, decay, initial, reset, reverse, rate);
    check_no_tangents(x, recur, input, decay, initial);
    const at::NoGradGuard no_grad;
    const RecurrenceResult r = run_recurrence(x, recur, input, decay, initial, reset, reverse, rate, false);
    return {r.y, r.last};
}

at::Tensor gated_recurrence_step(const at::Tensor &x, const at::Tensor &recur,
                                 const at::Tensor &input, const at::Tensor &decay,
                                 const at::Tensor &state, double rate) {
    check_recurrence_inputs(x, recur, input, decay, 2, "[batch, channels]");
    check_state(state, "state", x);
    TORCH_CHECK(state.is_contiguous(), "`state` is updated in place and has to be contiguous");
    TORCH_CHECK(!(state.requires_grad() && torch::autograd::GradMode::is_enabled()),
                "`state` is updated in place and cannot require a gradient");
    check_no_tangents(x, recur, input, decay, state);
    const c10::DeviceGuard guard(x.device());
    const at::NoGradGuard no_grad;
    const RecurrenceInputs in{dense_rows(x), dense_rows(recur), dense_rows(input),
                              of_type(decay, at::kFloat).contiguous(), {}, {}};
    const pesq_recurrence p = in.call(false, rate);
    at::Tensor y = at::empty(x.sizes(), x.options());
    check(pesq_recurrence_step(&p, state.data_ptr<float>(), y.data_ptr(), current_stream(x)),
          "pesq_recurrence_step");
    written(state);
    return y;
}

// ---------------------------------------------------------------------------
// residual norm
// ---------------------------------------------------------------------------

// [..., channels] as rows of neighbours: t itself where its rows are evenly spaced
at::Tensor as_rows(const at::Tensor &t, int64_t rows, int64_t channels) {
    return dense_rows(t.dim() == 2 ? t : t.reshape({rows, channels}));
}

struct NormInputs {
    at::Tensor x, branch, gate, post, scale, next;

    pesq_residual_norm call(double eps) const {
        pesq_residual_norm p{};
        const at::Tensor &typed = branch.defined() ? branch : x;
        p.rows = x.size(0);
        p.channels = x.size(1);
        p.stream_dtype = type_code(x, "`x`");
        p.dtype = type_code(typed, "`branch`");
        p.eps = eps;
        const std::array<const at::Tensor *, 3> operands{&x, &branch, &gate};
        for (int k = 0; k < 3; ++k) {
            p.strides[k] = operands[k]->defined() ? operands[k]->stride(0) : 0;
        }
        p.x = x.data_ptr();
        p.branch = data(branch);
        p.gate = data(gate);
        p.post_weight = data_or_null<float>(post);
        p.scale = data_or_null<float>(scale);
        p.next_weight = data_or_null<float>(next);
        return p;
    }
};

struct NormResult {
    NormInputs in;
    int32_t dtype;
    at::Tensor inverse;
    variable_list out;  // [x_out][n_out]
};

// dtype: of n where there is no branch; keep: with what the backward reads
NormResult run_norm(const at::Tensor &x, const OptTensor &branch, const OptTensor &gate,
                    const OptTensor &post, const OptTensor &scale, const OptTensor &next,
                    int64_t dtype, double eps, bool keep) {
    const c10::DeviceGuard guard(x.device());
    const int64_t channels = x.size(-1), rows = channels ? x.numel() / channels : 0;
    const auto rows_of = [&](const OptTensor &t) {
        return t ? as_rows(*t, rows, channels) : at::Tensor();
    };
    const auto weight = [](const OptTensor &t) { return t ? t->contiguous() : at::Tensor(); };
    NormResult r;
    r.in = {rows_of(x), rows_of(branch), rows_of(gate), weight(post), weight(scale), weight(next)};
    pesq_residual_norm p = r.in.call(eps);
    if (!branch) p.dtype = static_cast<int32_t>(dtype);
    r.dtype = p.dtype;
    const at::ScalarType typed = p.dtype == PESQ_F32    ? at::kFloat
                                 : p.dtype == PESQ_BF16 ? at::kBFloat16
                                                        : at::kHalf;
    at::Tensor x_out, n_out;
    if (branch) r.out.push_back(x_out = at::empty(x.sizes(), x.options()));
    if (next) r.out.push_back(n_out = at::empty(x.sizes(), x.options().dtype(typed)));
    if (keep) r.inverse = at::empty({rows, 2}, x.options().dtype(at::kFloat));
    check(pesq_residual_norm_forward(&p, data(x_out), data(n_out), data_or_null<float>(r.inverse),
                                     current_stream(x)),
          "pesq_residual_norm_forward");
    return r;
}

struct ResidualNorm : public torch::autograd::Function<ResidualNorm> {
    // variables: x, branch, gate, post, scale, next
    static variable_list forward(AutogradContext *ctx, const at::Tensor &x, const OptTensor &branch,
                                 const OptTensor &gate, const OptTensor &post,
                                 const OptTensor &scale, const OptTensor &next, int64_t dtype,
                                 double eps) {
        const NormResult r = run_norm(x, branch, gate, post, scale, next, dtype, eps, true);
        ctx->set_materialize_grads(false);
        ctx->save_for_backward({r.in.x, r.in.branch, r.in.gate, r.in.post, r.in.scale, r.in.next, r.inverse});
        ctx->saved_data["eps"] = eps;
        const at::Tensor none;
        const auto operand = [&](const OptTensor &t) { return t ? &*t : &none; };
        ctx->saved_data["requiring"] =
            requiring<6>({&x, operand(branch), operand(gate), operand(post), operand(scale), operand(next)});
        ctx->saved_data["dtype"] = static_cast<int64_t>(r.dtype);
        ctx->saved_data["sizes"] = x.sizes().vec();
        return r.out;
    }

    static variable_list backward(AutogradContext *ctx, variable_list grads) {
        variable_list out(8);  // one per argument of forward
        const variable_list saved = ctx->get_saved_variables();
        const NormInputs in{saved[0], saved[1], saved[2], saved[3], saved[4], saved[5]};
        at::Tensor g_x_out, g_n_out;
        if (in.branch.defined()) g_x_out = grads[0];
        if (in.next.defined()) g_n_out = grads.back();
        if (!g_x_out.defined() && !g_n_out.defined()) return out;
        const c10::DeviceGuard guard(in.x.device());
        pesq_residual_norm p = in.call(ctx->saved_data["eps"].toDouble());
        p.dtype = static_cast<int32_t>(ctx->saved_data["dtype"].toInt());
        const auto sizes = ctx->saved_data["sizes"].toIntVector();
        {
            const at::NoGradGuard no_grad;
            if (g_x_out.defined()) {
                g_x_out = as_rows(of_type(g_x_out, in.x.scalar_type()), p.rows, p.channels);
            }
            if (g_n_out.defined()) g_n_out = as_rows(g_n_out, p.rows, p.channels);
        }
        size_t bytes = 0;
        check(pesq_residual_norm_workspace(&p, &bytes), "pesq_residual_norm_workspace");
        at::Tensor ws = at::empty({static_cast<int64_t>(bytes)}, in.x.options().dtype(at::kByte));
        // variables that are there are numbered in order
        const std::array<const at::Tensor *, 6> operands{&in.x,    &in.branch, &in.gate,
                                                         &in.post, &in.scale,  &in.next};
        int variable = 0;
        for (int k = 0; k < 6; ++k) {
            if (!operands[k]->defined() || !ctx->needs_input_grad(variable++)) continue;
            if (k < 3) {
                out[k] = at::empty(sizes, operands[k]->options());
            } else {
                out[k] = at::empty({p.channels}, operands[k]->options());
            }
        }
        at::Tensor g_next = out[5];
        if (g_next.defined() && !g_n_out.defined()) {
            g_next.zero_();
            g_next = at::Tensor();
        }
        const std::array<int64_t, 2> strides{g_x_out.defined() ? g_x_out.stride(0) : 0,
                                             g_n_out.defined() ? g_n_out.stride(0) : 0};
        check(pesq_residual_norm_backward(
                  &p, data(g_x_out), data(g_n_out), strides.data(), data_or_null<float>(saved[6]),
                  data(out[0]), data(out[1]), data(out[2]), data_or_null<float>(out[3]),
                  data_or_null<float>(out[4]), data_or_null<float>(g_next), data(ws),
                  current_stream(in.x)),
              "pesq_residual_norm_backward");
        // x' alone is linear in x, the scale and the weight
        constexpr int64_t kX = 1, kBranch = 2, kGate = 4, kPost = 8, kScale = 16, kNext = 32;
        constexpr int64_t kOfY = kBranch | kGate, kAll = kX | kOfY | kPost | kScale | kNext;
        const int64_t of_n = g_n_out.defined() ? kAll : 0;
        mark_once<6>(out, grads, ctx->saved_data["requiring"].toInt(),
                     {of_n, of_n | kOfY | kPost | kScale, of_n | kOfY | kPost | kScale, of_n | kOfY | kScale,
                      of_n | kOfY | kPost, of_n & ~kNext});
        return out;
    }
};

void check_weight(const OptTensor &w, const char *name, const at::Tensor &x) {
    if (!w) return;
    check_gpu(*w, name, x);
    TORCH_CHECK(w->is_floating_point() && w->dim() == 1 && w->size(0) == x.size(-1), "`", name,
                "` has to be a floating [channels] tensor, got ", w->scalar_type(), " ", w->sizes());
}

// (x, branch, post, gate, scale, next, dtype of n without a branch) -> [x_out][n_out]
std::vector<at::Tensor> residual_norm(const at::Tensor &x, const OptTensor &branch,
                                      const OptTensor &post, const OptTensor &gate,
                                      const OptTensor &scale, const OptTensor &next, double eps,
                                      std::optional<at::ScalarType> dtype) {
    TORCH_CHECK(x.is_cuda(), "The HIP backend needs `x` to live on a GPU.");
    TORCH_CHECK(x.dim() >= 1, "the residual norm expects [..., channels], got a scalar");
    type_code(x, "`x`");
    const std::array<std::pair<const char *, const OptTensor *>, 2> rows{
        {{"branch", &branch}, {"gate", &gate}}};
    for (const auto &[name, t] : rows) {
        if (!*t) continue;
        check_gpu(**t, name, x);
        TORCH_CHECK((*t)->sizes() == x.sizes(), "`", name, "` has to have the shape of x, ",
                    x.sizes(), ", got ", (*t)->sizes());
        type_code(**t, name);
        TORCH_CHECK((*t)->scalar_type() == branch->scalar_type(), "`gate` has to have the type of "
                    "the branch, ", branch->scalar_type(), ", got ", (*t)->scalar_type());
    }
    int64_t code = 0;
    const at::ScalarType typed = branch ? branch->scalar_type() : dtype.value_or(x.scalar_type());
    TORCH_CHECK(x.scalar_type() == at::kFloat || x.scalar_type() == typed, "`x` has to be float32 or "
                "of the type ", typed, ", got ", x.scalar_type());
    if (!branch) {
        TORCH_CHECK(typed == at::kFloat || typed == at::kBFloat16 || typed == at::kHalf,
                    "the result has to be float32, bfloat16 or float16, got ", typed);
        code = typed == at::kFloat ? PESQ_F32 : typed == at::kBFloat16 ? PESQ_BF16 : PESQ_F16;
    }
    check_weight(post, "weight", x);
    check_weight(scale, "scale", x);
    check_weight(next, branch ? "next_weight" : "weight", x);
    const auto f32 = [](const OptTensor &t) { return t ? OptTensor(of_type(*t, at::kFloat)) : t; };
    const OptTensor w = f32(post), s = f32(scale), n = f32(next);
    bool keep = x.requires_grad();
    for (const OptTensor *t : std::array<const OptTensor *, 5>{&branch, &gate, &w, &s, &n}) {
        keep = keep || (*t && (*t)->requires_grad());
    }
    if (keep && torch::autograd::GradMode::is_enabled()) {
        return ResidualNorm::apply(x, branch, gate, w, s, n, code, eps);
    }
    check_no_tangents(x, branch, gate, w, s, n);
    const at::NoGradGuard no_grad;
    return run_norm(x, branch, gate, w, s, n, code, eps, false).out;
}

// ---------------------------------------------------------------------------
// AdamW
// ---------------------------------------------------------------------------

// The parameters of one optimizer, the place of each in the moments' arrays,
// and these arrays.  Gradients are taken from the parameters at each step.
bool capturing(const c10::Device &device) {
    hipStreamCaptureStatus status = hipStreamCaptureStatusNone;
    const hipError_t error = hipStreamIsCapturing(c10::hip::getCurrentHIPStream(device.index()).stream(), &status);
    if (error == hipErrorStreamCaptureImplicit) {  // the default stream, while another one is captured
        (void)hipGetLastError();
        return false;
    }
    TORCH_CHECK(error == hipSuccess, "hipStreamIsCapturing: ", hipGetErrorString(error));
    return status != hipStreamCaptureStatusNone;
}

class AdamWPlan {
  public:
    static constexpr int64_t kBlock = 256;

    AdamWPlan(std::vector<std::vector<at::Tensor>> groups, int64_t bits)
        : groups_(std::move(groups)), bits_(bits) {
        TORCH_CHECK(bits == 32 || bits == 8, "moments have 32 or 8 bits, got ", bits);
        at::TensorOptions options;
        for (const auto &group : groups_) {
            first_.emplace_back();
            counts_.emplace_back();
            for (const at::Tensor &p : group) {
                TORCH_CHECK(p.is_cuda(), "HipAdamW needs its parameters to live on a GPU.");
                if (!options.has_device()) options = options.device(p.device());
                TORCH_CHECK(p.device() == options.device(), "HipAdamW needs all parameters on one GPU.");
                type_code(p, "a parameter");
                first_.back().push_back(total_);
                counts_.back().push_back(p.numel());
                total_ += (p.numel() + kBlock - 1) / kBlock * kBlock;
                ++tensors_;
            }
        }
        if (tensors_ == 0) {
            steps_ = at::zeros({0}, at::kLong);
            return;
        }
        const c10::DeviceGuard guard(options.device());
        TORCH_CHECK(!capturing(options.device()), "HipAdamW lays its moments out at its first step, which cannot be "
                    "captured in a graph: take one before, or call `moments()`.");
        // (pinned: the GPU counts in it once a step was captured)
        steps_ = at::zeros({tensors_}, at::TensorOptions().dtype(at::kLong).pinned_memory(true));
        corrections_ = at::empty({tensors_, 2}, options.dtype(at::kFloat));
        const auto type = [&](at::ScalarType t) { return options.dtype(t); };
        if (bits == 32) {
            arrays_ = {at::zeros({total_}, type(at::kFloat)), at::zeros({total_}, type(at::kFloat))};
        } else {
            arrays_ = {at::zeros({total_}, type(at::kChar)), at::zeros({total_}, type(at::kByte)),
                       at::zeros({total_ / kBlock}, type(at::kFloat)),
                       at::zeros({total_ / kBlock}, type(at::kFloat))};
        }
    }

    // [m, v] or [m, v, scales of m, scales of v] of parameter k of a group, as views
    std::vector<at::Tensor> views(int64_t group, int64_t k) const {
        const at::Tensor &p = groups_.at(group).at(k);
        const int64_t first = first_[group][k], count = counts_[group][k];
        std::vector<at::Tensor> out;
        for (size_t n = 0; n < arrays_.size(); ++n) {
            if (n < 2) {
                out.push_back(arrays_[n].narrow(0, first, count).view(p.sizes()));
            } else {
                out.push_back(arrays_[n].narrow(0, first / kBlock, (count + kBlock - 1) / kBlock));
            }
        }
        return out;
    }

    at::Tensor steps() const { return steps_; }

    // `state` and `groups` are what the plan stands for: see `current`.
    void watch(const pybind11::dict &state, const pybind11::list &groups) {
        entries_.clear();
        params_.clear();
        for (const auto &group : groups) {
            params_.emplace_back();
            for (const auto &p : pybind11::reinterpret_borrow<pybind11::dict>(group)["params"]) {
                params_.back().push_back(pybind11::reinterpret_borrow<pybind11::object>(p));
            }
        }
        for (const auto &[key, held] : state) {
            Entry entry{pybind11::reinterpret_borrow<pybind11::object>(key),
                        pybind11::reinterpret_borrow<pybind11::object>(held), {}};
            if (PyDict_Check(held.ptr())) {
                for (const auto &item : pybind11::reinterpret_borrow<pybind11::dict>(held)) {
                    entry.values.push_back(pybind11::reinterpret_borrow<pybind11::object>(item.second));
                }
            }
            entries_.push_back(std::move(entry));
        }
    }

    // Whether the optimizer's state and groups are those that the plan was made
    // from: by the identity of every entry, tensor and parameter, in order (through
    // the interpreter's own interface: a few nanoseconds each, in every step).
    bool current(const pybind11::dict &state, const pybind11::list &groups) const {
        if (static_cast<size_t>(PyDict_Size(state.ptr())) != entries_.size() || !same_groups(groups)) return false;
        Py_ssize_t at = 0;
        PyObject *key, *held, *value;
        for (const Entry &entry : entries_) {
            if (!PyDict_Next(state.ptr(), &at, &key, &held) || key != entry.key.ptr() || held != entry.held.ptr()) {
                return false;
            }
            if (!PyDict_Check(held)) continue;
            if (static_cast<size_t>(PyDict_Size(held)) != entry.values.size()) return false;
            Py_ssize_t inner = 0;
            for (const pybind11::object &kept : entry.values) {
                if (!PyDict_Next(held, &inner, nullptr, &value) || value != kept.ptr()) return false;
            }
        }
        return true;
    }

    bool same_groups(const pybind11::list &groups) const {
        if (groups.size() != params_.size()) return false;
        static PyObject *const name = PyUnicode_InternFromString("params");
        for (size_t g = 0; g < params_.size(); ++g) {
            PyObject *group = PyList_GET_ITEM(groups.ptr(), static_cast<Py_ssize_t>(g));
            PyObject *params = PyDict_Check(group) ? PyDict_GetItem(group, name) : nullptr;
            if (!params || !PyList_Check(params)) return false;
            if (static_cast<size_t>(PyList_GET_SIZE(params)) != params_[g].size()) return false;
            for (size_t k = 0; k < params_[g].size(); ++k) {
                if (PyList_GET_ITEM(params, static_cast<Py_ssize_t>(k)) != params_[g][k].ptr()) return false;
            }
        }
        return true;
    }

    // Whether a step was captured in a graph.  From then on the GPU keeps the counts,
    // the captured steps' and all others', and the plan's memory is the graph's.
    bool captured() const { return captured_; }

    void step(int64_t group, double lr, double beta1, double beta2, double eps,
              double weight_decay) {
        struct Bucket {
            pesq_adamw_options options;
            std::vector<pesq_adamw_tensor> tensors;
            std::vector<int64_t *> steps;
        };
        std::vector<Bucket> buckets;  // parameters of one type and, where the host counts, step count
        std::vector<size_t> stepped;
        std::vector<at::Tensor> copies;
        int64_t at_step = 0;
        for (int64_t g = 0; g < group; ++g) at_step += static_cast<int64_t>(groups_.at(g).size());
        int64_t *steps = steps_.data_ptr<int64_t>() + at_step;
        const auto &params = groups_.at(group);
        const auto &firsts = first_[group], &counts = counts_[group];
        const c10::Device device = tensors_ > 0 ? arrays_[0].device() : c10::Device(c10::kCPU);
        if (tensors_ > 0 && !captured_ && capturing(device)) {
            captured_ = true;
            // A graph may count after the optimizer is gone, and nothing tells the allocator of pinned
            // memory: the counts stay where they are until the process ends.
            new at::Tensor(steps_);
        }
        stepped.reserve(params.size());
        for (size_t k = 0; k < params.size(); ++k) {
            const at::Tensor &p = params[k], &grad = p.grad();
            if (!grad.defined()) continue;
            TORCH_CHECK(p.numel() == counts[k] && p.is_contiguous() && p.device() == device,
                        "HipAdamW needs contiguous parameters that keep their size and GPU.");
            TORCH_CHECK(grad.layout() == at::kStrided && grad.scalar_type() == p.scalar_type() &&
                            grad.sizes() == p.sizes() && grad.device() == device,
                        "HipAdamW needs dense gradients of the parameters' type and GPU.");
            if (!grad.is_contiguous()) copies.push_back(grad.contiguous());
            const void *from = (grad.is_contiguous() ? grad : copies.back()).data_ptr();
            const int32_t dtype = type_code(p, "a parameter");
            Bucket *bucket = nullptr;
            for (Bucket &b : buckets) {
                if (b.options.dtype == dtype && (captured_ || b.options.step == steps[k] + 1)) bucket = &b;
            }
            if (!bucket) {
                buckets.push_back({{dtype, static_cast<int32_t>(bits_), captured_ ? 0 : steps[k] + 1, lr, beta1,
                                    beta2, eps, weight_decay}, {}, {}});
                bucket = &buckets.back();
                bucket->tensors.reserve(params.size());
            }
            bucket->tensors.push_back({p.data_ptr(), from, counts[k], firsts[k]});
            if (captured_) bucket->steps.push_back(steps + k);
            stepped.push_back(k);
        }
        if (buckets.empty()) return;
        const c10::DeviceGuard guard(arrays_[0].device());
        const bool eight = bits_ == 8;
        float *m_scale = eight ? arrays_[2].data_ptr<float>() : nullptr;
        float *v_scale = eight ? arrays_[3].data_ptr<float>() : nullptr;
        float *corrections = corrections_.data_ptr<float>() + 2 * at_step;
        for (const Bucket &b : buckets) {
            const int64_t count = static_cast<int64_t>(b.tensors.size());
            if (captured_) {
                check(pesq_adamw_step_counted(b.tensors.data(), count, &b.options, b.steps.data(), corrections,
                                              arrays_[0].data_ptr(), arrays_[1].data_ptr(), m_scale, v_scale,
                                              current_stream(arrays_[0])),
                      "pesq_adamw_step_counted");
                corrections += 2 * count;
            } else {
                check(pesq_adamw_step(b.tensors.data(), count, &b.options, arrays_[0].data_ptr(),
                                      arrays_[1].data_ptr(), m_scale, v_scale, current_stream(arrays_[0])),
                      "pesq_adamw_step");
            }
        }
        for (const size_t k : stepped) {
            if (!captured_) ++steps[k];
            written(params[k]);
        }
    }

    // [m, v] as float32 arrays: the state's own with 32 bits
    std::vector<at::Tensor> moments() const {
        if (bits_ == 32 || arrays_.empty()) return arrays_;
        const c10::DeviceGuard guard(arrays_[0].device());
        const auto f32 = arrays_[2].options();
        std::vector<at::Tensor> out{at::empty({total_}, f32), at::empty({total_}, f32)};
        check(pesq_adamw_moments(arrays_[0].data_ptr(), arrays_[1].data_ptr(),
                                 arrays_[2].data_ptr<float>(), arrays_[3].data_ptr<float>(), total_,
                                 out[0].data_ptr<float>(), out[1].data_ptr<float>(),
                                 current_stream(arrays_[0])),
              "pesq_adamw_moments");
        return out;
    }

    int64_t first(int64_t group, int64_t k) const { return first_.at(group).at(k); }

  private:
    struct Entry {
        pybind11::object key, held;
        std::vector<pybind11::object> values;
    };

    std::vector<Entry> entries_;  // of the state
    std::vector<std::vector<pybind11::object>> params_;
    std::vector<std::vector<at::Tensor>> groups_;
    int64_t bits_, total_ = 0, tensors_ = 0;
    std::vector<std::vector<int64_t>> first_, counts_;
    at::Tensor steps_, corrections_;
    std::vector<at::Tensor> arrays_;
    bool captured_ = false;
};

}  // namespace

void bind_network(pybind11::module_ &m) {
    using pybind11::arg;
    m.def("gated_recurrence", &gated_recurrence,
          "(x, recur_gate, input_gate, decay, initial, reset, reverse, rate) -> [y, last]", arg("x"),
          arg("recur_gate"), arg("input_gate"), arg("decay"), arg("initial"), arg("reset"),
          arg("reverse"), arg("rate"));
    m.def("gated_recurrence_step", &gated_recurrence_step,
          "(x, recur_gate, input_gate, decay, state, rate) -> y, the state updated in place",
          arg("x"), arg("recur_gate"), arg("input_gate"), arg("decay"), arg("state"), arg("rate"));
    m.def(
        "residual_norm",
        [](const at::Tensor &x, const OptTensor &branch, const OptTensor &post, const OptTensor &gate,
           const OptTensor &scale, const OptTensor &next, double eps, const pybind11::object &dtype) {
            std::optional<at::ScalarType> type;
            if (!dtype.is_none()) type = torch::python::detail::py_object_to_dtype(dtype);
            return residual_norm(x, branch, post, gate, scale, next, eps, type);
        },
        "(x, branch, weight, gate, scale, next_weight, eps, dtype) -> [x_out][n_out]", arg("x"),
        arg("branch"), arg("weight"), arg("gate"), arg("scale"), arg("next_weight"), arg("eps"),
        arg("dtype"));
    pybind11::class_<AdamWPlan>(m, "AdamWPlan", "the tensors and moments of one optimizer")
        .def(pybind11::init<std::vector<std::vector<at::Tensor>>, int64_t>(), arg("groups"),
             arg("bits"))
        .def("step", &AdamWPlan::step, arg("group"), arg("lr"), arg("beta1"), arg("beta2"),
             arg("eps"), arg("weight_decay"))
        .def("views", &AdamWPlan::views)
        .def("first", &AdamWPlan::first)
        .def("steps", &AdamWPlan::steps)
        .def("watch", &AdamWPlan::watch)
        .def("current", &AdamWPlan::current)
        .def("same_groups", &AdamWPlan::same_groups)
        .def("captured", &AdamWPlan::captured)
        .def("moments", &AdamWPlan::moments);
}
