"""Host side checks of the network operators' C entry points: refusals before any
GPU work, workspace sizes, calls without elements; and the package's refusals of
host tensors.  No kernel is launched."""

import ctypes
import re

import pytest
import torch

from torch_pesq import _lib
from torch_pesq.hip_ops.adamw import HipAdamW
from torch_pesq.hip_ops.norm import pre_norm, residual_norm
from torch_pesq.hip_ops.recurrence import HipGatedRecurrence, gated_recurrence, gated_recurrence_step

ANY = 4096  # an address that is never read


def _message():
    return _lib.library().pesq_last_error().decode()


def _recurrence(**changes):
    p = _lib.Recurrence(batch=2, time=10, channels=8, rate=8.0, x=ANY, recur_gate=ANY, input_gate=ANY, decay=ANY)
    for name, value in changes.items():
        setattr(p, name, value)
    return p


@pytest.mark.parametrize("changes,message", [
    ({"dtype": 3}, "element type"), ({"batch": -1}, "sizes"), ({"batch": 65536}, "65535"),
    ({"channels": 2**24 + 1}, "2\\^24"), ({"time": 2**33}, "2\\^32"), ({"rate": 0.0}, "rate"),
    ({"rate": float("nan")}, "rate"), ({"rate": float("inf")}, "rate"),
])
def test_recurrence_refuses(changes, message):
    lib, p, size = _lib.library(), _recurrence(**changes), ctypes.c_size_t()
    for status in (lib.pesq_recurrence_workspace(p, size, size, size),
                   lib.pesq_recurrence_forward(p, ANY, ANY, None, ANY, None),
                   lib.pesq_recurrence_backward(p, None, None, None, ANY, None, None, None, None, None, ANY, None)):
        assert status == _lib.ERR_ARGUMENT
        assert re.search(message, _message())


@pytest.mark.parametrize("rate,status", [(2.0**126, 0), (1e-30, 0), (2.0**127, 1), (1e39, 1)])
def test_recurrence_rates_fit_float32(rate, status):
    """The kernels hold the rate times log2(e) in float32, where 1e39 would be infinite
    and the product with a softplus of 0 a NaN."""

    assert _lib.library().pesq_recurrence_workspace(_recurrence(rate=rate), None, None, None) == status
    assert status == 0 or "rate" in _message()
    if status:
        with pytest.raises(ValueError, match="rate"):
            HipGatedRecurrence(4, rate=rate)
    else:
        HipGatedRecurrence(4, rate=rate)


def test_recurrence_null_arguments_and_strides():
    lib = _lib.library()
    for name in ("x", "recur_gate", "input_gate", "decay"):
        assert lib.pesq_recurrence_forward(_recurrence(**{name: None}), ANY, None, None, ANY, None) == 1
    assert lib.pesq_recurrence_forward(_recurrence(), None, None, None, ANY, None) == 1
    p = _recurrence()
    p.strides[2][1] = 2**26
    assert lib.pesq_recurrence_forward(p, ANY, None, None, ANY, None) == 1 and "apart" in _message()
    p = _recurrence()
    p.strides[1][0] = -8
    assert lib.pesq_recurrence_forward(p, ANY, None, None, ANY, None) == 1 and "negative stride" in _message()
    assert lib.pesq_recurrence_backward(_recurrence(), ANY, None, None, ANY, None, None, None, None, None, ANY, None) == 1
    assert "strides" in _message()
    assert lib.pesq_recurrence_step(_recurrence(), ANY, ANY, None) == 1 and "one frame" in _message()
    assert lib.pesq_recurrence_forward(None, ANY, None, None, ANY, None) == 1
    # nothing to do: no pointer is needed
    for empty in ({"batch": 0}, {"channels": 0}):
        p = _recurrence(x=None, recur_gate=None, input_gate=None, decay=None, **empty)
        assert lib.pesq_recurrence_forward(p, None, None, None, None, None) == 0


def test_recurrence_workspaces_follow_the_sizes():
    lib = _lib.library()
    sizes = [ctypes.c_size_t() for _ in range(3)]
    for time in (0, 1, 16, 17, 4000):
        p = _recurrence(time=time)
        assert lib.pesq_recurrence_workspace(p, *sizes) == 0
        # float32 states before every few steps
        assert sizes[0].value % (2 * 8 * 4) == 0 and sizes[0].value // (2 * 8 * 4) <= -(-time // 8)
        # the joining needs no scratch where one workgroup takes a whole row
        assert (sizes[1].value > 0) == (time > 64)


def _norm(**changes):
    p = _lib.ResidualNorm(rows=3, channels=16, eps=1e-6, x=ANY, branch=ANY, gate=ANY, post_weight=ANY, scale=ANY,
                          next_weight=ANY)
    for name, value in changes.items():
        setattr(p, name, value)
    return p


@pytest.mark.parametrize("changes,message", [
    ({"dtype": 7}, "element type"), ({"dtype": 1, "stream_dtype": 2}, "stream's type"), ({"rows": -1}, "rows"),
    ({"rows": 2**31}, "rows"), ({"channels": 0}, "channels"), ({"channels": 8193}, "channels"),
    ({"eps": -1.0}, "eps"), ({"eps": float("nan")}, "eps"), ({"post_weight": None}, "its weight"),
    ({"branch": None}, "only the next weight"), ({"x": None}, "null"),
])
def test_residual_norm_refuses(changes, message):
    lib, p = _lib.library(), _norm(**changes)
    strides = (ctypes.c_int64 * 2)(16, 16)
    assert lib.pesq_residual_norm_forward(p, ANY, ANY, None, None) == 1 and message in _message()
    assert lib.pesq_residual_norm_backward(p, ANY, ANY, strides, ANY, ANY, ANY, ANY, ANY, ANY, ANY, ANY, None) == 1
    assert message in _message()


def test_residual_norm_outputs_and_gradients_that_are_not_there():
    lib = _lib.library()
    strides = (ctypes.c_int64 * 2)(16, 16)
    assert lib.pesq_residual_norm_forward(_norm(), None, ANY, None, None) == 1
    assert lib.pesq_residual_norm_forward(_norm(), ANY, None, None, None) == 1
    p = _norm(gate=None)
    assert lib.pesq_residual_norm_backward(p, ANY, ANY, strides, ANY, ANY, ANY, ANY, None, None, None, ANY, None) == 1
    assert "not there" in _message()
    p = _norm(next_weight=None)
    assert lib.pesq_residual_norm_backward(p, ANY, ANY, strides, ANY, ANY, None, None, None, None, None, ANY, None) == 1
    assert lib.pesq_residual_norm_forward(_norm(rows=0, x=None, branch=None), None, None, None, None) == 0


def test_adamw_refuses():
    lib = _lib.library()
    good = {"dtype": 0, "state_bits": 32, "step": 1, "lr": 1e-3, "beta1": 0.9, "beta2": 0.999, "eps": 1e-8}
    tensors = (_lib.AdamwTensor * 1)(_lib.AdamwTensor(ANY, ANY, 100, 0))

    def call(tensors=tensors, count=1, arrays=(ANY, ANY, ANY, ANY), **changes):
        return lib.pesq_adamw_step(tensors, count, _lib.AdamwOptions(**dict(good, **changes)), *arrays, None)

    for changes, message in (({"dtype": 5}, "element type"), ({"state_bits": 16}, "32 or 8"), ({"step": 0}, "from 1"),
                             ({"beta1": 1.0}, "betas"), ({"beta2": -0.5}, "betas")):
        assert call(**changes) == 1 and message in _message()
    assert call(arrays=(ANY, None, ANY, ANY)) == 1
    assert call(arrays=(ANY, ANY, None, ANY), state_bits=8) == 1
    assert call(tensors=(_lib.AdamwTensor * 1)(_lib.AdamwTensor(ANY, ANY, 100, 100))) == 1
    assert call(tensors=(_lib.AdamwTensor * 1)(_lib.AdamwTensor(ANY, ANY, -1, 0))) == 1
    assert call(tensors=(_lib.AdamwTensor * 1)(_lib.AdamwTensor(ANY, None, 10, 0))) == 1
    assert call(tensors=None) == 1
    # nothing to do
    assert call(tensors=None, count=0) == 0
    assert call(tensors=(_lib.AdamwTensor * 1)(_lib.AdamwTensor(None, None, 0, 256))) == 0
    assert lib.pesq_adamw_moments(ANY, ANY, ANY, ANY, 100, ANY, ANY, None) == 1
    assert lib.pesq_adamw_moments(None, None, None, None, 0, None, None, None) == 0


def test_host_tensors_are_refused():
    x, w = torch.zeros(2, 5, 8), torch.zeros(8)
    for call in (lambda: gated_recurrence(x, x, x, w), lambda: gated_recurrence_step(x[0], x[0], x[0], w, x[0]),
                 lambda: HipGatedRecurrence(8)(x, x, x), lambda: residual_norm(x, x, w), lambda: pre_norm(x, w)):
        with pytest.raises(RuntimeError, match="live on a GPU"):
            call()
    p = torch.nn.Parameter(torch.zeros(4))
    p.grad = torch.zeros(4)
    with pytest.raises(RuntimeError, match="live on a GPU"):
        HipAdamW([p]).step()


def test_optimizer_options():
    p, q = (torch.nn.Parameter(torch.zeros(4)) for _ in range(2))
    with pytest.raises(ValueError, match="same `state_bits`"):
        HipAdamW([{"params": [p]}, {"params": [q], "state_bits": 8}])
    opt = HipAdamW([p], state_bits=8)
    assert opt.state_bits == 8 and opt.state_dict()["param_groups"][0]["state_bits"] == 8


@pytest.mark.parametrize("options,message", [
    ({"lr": -1.0}, "learning rate"), ({"betas": (0.9, 1.0)}, "betas"), ({"eps": -1.0}, "eps"), ({"state_bits": 32}, "same"),
])
def test_a_refused_group_is_not_added(options, message):
    p, q = (torch.nn.Parameter(torch.zeros(4)) for _ in range(2))
    opt = HipAdamW([p], state_bits=8)
    with pytest.raises(ValueError, match=message):
        opt.add_param_group({"params": [q], **options})
    assert [g["params"] for g in opt.param_groups] == [[p]]
    with pytest.raises(ValueError, match="32 or 8"):
        HipAdamW([{"params": [q], "state_bits": 16}])
    assert HipAdamW([{"params": [q], "state_bits": 8}]).state_bits == 8
    opt.add_param_group({"params": [q], "lr": 0.5})
    assert opt.param_groups[1]["lr"] == 0.5 and opt.param_groups[1]["state_bits"] == 8


def test_module_decay_spans_the_asked_memory():
    module = HipGatedRecurrence(1000, rate=4.0, fastest=0.5, slowest=0.99)
    open_gate = torch.exp(-4.0 * torch.nn.functional.softplus(module.decay.detach().double()))
    assert 0.4999 < float(open_gate.min()) < 0.52 and 0.97 < float(open_gate.max()) < 0.9901


@pytest.mark.parametrize("dtype,most", [(0, 2**25), (1, 2**26), (2, 2**26)])
def test_recurrence_steps_apart_in_bytes(dtype, most):
    """The byte offset of a part's last row, 15 steps from its first, stays below 2^31."""

    lib, size = _lib.library(), ctypes.c_size_t()
    assert 15 * (most - 1) * (2 if dtype else 4) < 2**31
    for tensor in range(3):
        p = _recurrence(dtype=dtype)
        p.strides[tensor][1] = most - 1
        assert lib.pesq_recurrence_workspace(p, size, size, size) == 0
        p.strides[tensor][1] = most
        assert lib.pesq_recurrence_workspace(p, size, size, size) == 1 and "apart" in _message()
    # the upstream gradient's
    p = _recurrence(dtype=dtype, batch=0)
    for stride, status in ((most - 1, 0), (most, 1)):
        strides = (ctypes.c_int64 * 2)(0, stride)
        assert lib.pesq_recurrence_backward(p, ANY, strides, None, ANY, None, None, None, None, ANY, ANY, None) == status


@pytest.mark.parametrize("bits", [8, 32])
def test_adamw_of_tensors_without_elements(bits):
    """Nothing to do: no address is needed, as such tensors have none."""

    options = _lib.AdamwOptions(dtype=0, state_bits=bits, step=1, lr=1e-3, beta1=0.9, beta2=0.999, eps=1e-8)
    tensors = (_lib.AdamwTensor * 2)()
    assert _lib.library().pesq_adamw_step(tensors, 2, options, None, None, None, None, None) == 0
    tensors[1] = _lib.AdamwTensor(param=ANY, grad=ANY, count=1, first=0)
    assert _lib.library().pesq_adamw_step(tensors, 2, options, None, None, None, None, None) == 1
    assert "null argument" in _message()


def test_adamw_counted_steps_refuse():
    """As the others, but for the number of the step, which is not theirs to give."""

    lib, tensors = _lib.library(), (_lib.AdamwTensor * 1)(_lib.AdamwTensor(ANY, ANY, 100, 0))
    good = {"dtype": 0, "state_bits": 32, "step": 0, "lr": 1e-3, "beta1": 0.9, "beta2": 0.999, "eps": 1e-8}
    steps = (ctypes.c_void_p * 1)(ANY)

    def call(count=1, steps=steps, corrections=ANY, arrays=(ANY, ANY, ANY, ANY), **changes):
        return lib.pesq_adamw_step_counted(tensors, count, _lib.AdamwOptions(**dict(good, **changes)), steps,
                                           corrections, *arrays, None)

    for changes, message in (({"steps": None}, "null"), ({"corrections": None}, "null"), ({"corrections": ANY + 4}, "8 bytes"),
                             ({"steps": (ctypes.c_void_p * 1)(None)}, "no count"), ({"beta1": 1.0}, "betas"),
                             ({"arrays": (ANY, None, ANY, ANY)}, "null"), ({"count": -1}, "null")):
        assert call(**changes) == 1 and message in _message(), changes
    # nothing to do
    assert call(count=0, steps=None, corrections=None) == 0


def test_adamw_moments_fit_a_launch():
    """Work items of a launch, four elements each in whole workgroups, stay below 2^32."""

    for count, message in ((2**34 - 256, "elements"), (2**34 - 1024, "null argument"), (2**34, "elements")):
        assert _lib.library().pesq_adamw_moments(None, None, None, None, count, None, None, None) == 1
        assert message in _message()
