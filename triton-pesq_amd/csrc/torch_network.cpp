// PyTorch autograd nodes and entry points of the operators of the networks
// that the loss trains, in C++ for the reason torch_autograd.cpp gives.
//
// Each entry point checks its tensors, allocates outputs and workspaces on the
// caller's device and enqueues the library's calls on PyTorch's current stream.

#include "torch_common.hpp"

#include <array>
#include <optional>
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

// the gradients, with a derivative that raises where a double backward would need one
void mark_once(variable_list &grads, const variable_list &upstream) {
    bool needed = false;
    for (const at::Tensor &g : upstream) needed = needed || (g.defined() && g.requires_grad());
    if (!needed || !torch::autograd::GradMode::is_enabled()) return;
    for (at::Tensor &g : grads) {
        if (g.defined()) g = OnceDifferentiable::apply(g.detach().requires_grad_(true));
    }
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
    TORCH_CHECK(decay.scalar_type() == at::kFloat && decay.dim() == 1 && decay.size(0) == x.size(-1),
                "`decay` has to be float32 [channels], got ", decay.scalar_type(), " ", decay.sizes());
}

void check_state(const at::Tensor &state, const char *name, const at::Tensor &x) {
    check_gpu(state, name, x);
    TORCH_CHECK(state.scalar_type() == at::kFloat && state.dim() == 2 &&
                    state.size(0) == x.size(0) && state.size(1) == x.size(-1),
                "`", name, "` has to be float32 [batch, channels], got ", state.scalar_type(), " ",
                state.sizes());
}

struct Recurrence : public torch::autograd::Function<Recurrence> {
    static variable_list forward(AutogradContext *ctx, const at::Tensor &x, const at::Tensor &recur,
                                 const at::Tensor &input, const at::Tensor &decay,
                                 const OptTensor &initial, const OptTensor &reset, bool reverse,
                                 double rate, bool keep) {
        const c10::DeviceGuard guard(x.device());
        RecurrenceInputs in{dense_rows(x), dense_rows(recur), dense_rows(input), decay.contiguous(),
                            initial ? initial->contiguous() : at::Tensor(),
                            reset ? reset->contiguous() : at::Tensor()};
        const pesq_recurrence p = in.call(reverse, rate);
        size_t starts_bytes = 0, ws_bytes = 0;
        check(pesq_recurrence_workspace(&p, &starts_bytes, &ws_bytes, nullptr),
              "pesq_recurrence_workspace");
        const auto bytes = x.options().dtype(at::kByte);
        at::Tensor starts, ws;
        if (keep) starts = at::empty({static_cast<int64_t>(starts_bytes)}, bytes);
        if (ws_bytes > 0) ws = at::empty({static_cast<int64_t>(ws_bytes)}, bytes);
        at::Tensor y = at::empty(x.sizes(), x.options());
        at::Tensor last = at::empty({x.size(0), x.size(2)}, x.options().dtype(at::kFloat));
        check(pesq_recurrence_forward(&p, y.data_ptr(), last.data_ptr<float>(),
                                      static_cast<float *>(data(starts)), data(ws), current_stream(x)),
              "pesq_recurrence_forward");
        ctx->set_materialize_grads(false);
        if (keep) {
            ctx->save_for_backward({in.x, in.recur, in.input, in.decay, in.initial, in.reset, starts});
            ctx->saved_data["reverse"] = reverse;
            ctx->saved_data["rate"] = rate;
        }
        return {y, last};
    }

    static variable_list backward(AutogradContext *ctx, variable_list grads) {
        variable_list out(9);
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
            if (grads[0].defined()) g_y = dense_rows(grads[0].to(x.scalar_type()));
            if (grads[1].defined()) g_last = grads[1].to(at::kFloat).contiguous();
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
        mark_once(out, grads);
        return out;
    }
};

std::vector<at::Tensor> gated_recurrence(const at::Tensor &x, const at::Tensor &recur,
                                         const at::Tensor &input, const at::Tensor &decay,
                                         const OptTensor &initial, const OptTensor &reset,
                                         bool reverse, double rate) {
    check_recurrence_inputs(x, recur, input, decay, 3, "[batch, time, channels]");
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
    return Recurrence::apply(x, recur, input, decay, initial, reset, reverse, rate, keep);
}

at::Tensor gated_recurrence_step(const at::Tensor &x, const at::Tensor &recur,
                                 const at::Tensor &input, const at::Tensor &decay,
                                 const at::Tensor &state, double rate) {
    check_recurrence_inputs(x, recur, input, decay, 2, "[batch, channels]");
    check_state(state, "state", x);
    TORCH_CHECK(state.is_contiguous(), "`state` is updated in place and has to be contiguous");
    const c10::DeviceGuard guard(x.device());
    const at::NoGradGuard no_grad;
    const RecurrenceInputs in{dense_rows(x), dense_rows(recur), dense_rows(input),
                              decay.contiguous(), {}, {}};
    const pesq_recurrence p = in.call(false, rate);
    at::Tensor y = at::empty(x.sizes(), x.options());
    check(pesq_recurrence_step(&p, state.data_ptr<float>(), y.data_ptr(), current_stream(x)),
          "pesq_recurrence_step");
    return y;
}

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
}
