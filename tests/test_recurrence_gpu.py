"""The gated linear recurrence against the formula in float64.

The reference walks the recurrence step by step on the CPU in float64 and
differentiates it with autograd.  Each step's factor a_t carries about four
float32 roundings (2.4e-7); over a memory of T steps they add up as a random
walk, so float32 results may be 1e-6 sqrt(T) of the largest value off (four
times the expected size), and 2e-6 for the element-wise parts; 16 bit results
half a unit of their type more.
"""

import math

import pytest
import torch
import torch.autograd.forward_ad as forward_ad

from torch_pesq.hip_ops.recurrence import HipGatedRecurrence, gated_recurrence, gated_recurrence_step

pytestmark = pytest.mark.gpu

HALF_UNIT = {torch.float32: 0.0, torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11}
NAMES = ("x", "recur", "input", "decay", "initial")


def _tolerance(dtype, steps):
    return HALF_UNIT[dtype] + 2e-6 + 1e-6 * math.sqrt(steps)


def _inputs(batch, time, channels, dtype, seed=0, resets=0.0, initial=True):
    g = torch.Generator().manual_seed(seed)
    t = {k: torch.randn(batch, time, channels, generator=g).to(dtype) for k in ("x", "recur", "input")}
    open_gate = 0.9 + 0.099 * torch.rand(channels, generator=g)
    t["decay"] = torch.log(torch.expm1(-torch.log(open_gate) / 8.0))
    t["initial"] = torch.randn(batch, channels, generator=g) if initial else None
    t["reset"] = torch.rand(batch, time, generator=g) < resets if resets else None
    t["g_y"] = torch.randn(batch, time, channels, generator=g).to(dtype)
    t["g_last"] = torch.randn(batch, channels, generator=g)
    return t


def _reference(t, reverse=False, rate=8.0, grads=True):
    """(y, last, gradients) in float64."""

    d = {k: None if t[k] is None else t[k].double().requires_grad_(grads) for k in NAMES}
    x = d["x"]
    batch, time, channels = x.shape
    u = rate * torch.nn.functional.softplus(d["decay"], threshold=60.0) * torch.sigmoid(d["recur"])
    a, s = torch.exp(-u), torch.sqrt(-torch.expm1(-2.0 * u))
    b = s * torch.sigmoid(d["input"]) * x
    h = d["initial"] if d["initial"] is not None else torch.zeros(batch, channels, dtype=torch.float64)
    ys = [None] * time
    for n in range(time):
        at = time - 1 - n if reverse else n
        if t["reset"] is not None:
            h = torch.where(t["reset"][:, at, None], torch.zeros_like(h), h)
        h = a[:, at] * h + b[:, at]
        ys[at] = h
    y = torch.stack(ys, 1) if time else x
    if not grads:
        return y, h, None
    names = [k for k in NAMES if d[k] is not None]
    loss = (y * t["g_y"].double()).sum() + (h * t["g_last"].double()).sum()
    return y.detach(), h.detach(), dict(zip(names, torch.autograd.grad(loss, [d[k] for k in names])))


def _run(t, reverse=False, rate=8.0, place=lambda v: v):
    d = {k: None if t[k] is None else place(t[k].cuda()).detach().requires_grad_() for k in NAMES}
    reset = None if t["reset"] is None else t["reset"].cuda()
    y, last = gated_recurrence(d["x"], d["recur"], d["input"], d["decay"], initial_state=d["initial"],
                               reset=reset, reverse=reverse, rate=rate)
    names = [k for k in NAMES if d[k] is not None]
    grads = torch.autograd.grad((y, last), [d[k] for k in names], (t["g_y"].cuda(), t["g_last"].cuda()))
    return y.detach(), last.detach(), dict(zip(names, grads))


def _close(got, want, tolerance, what):
    assert got.shape == want.shape, what
    if not want.numel():
        return
    got = got.double().cpu()
    assert torch.isfinite(got).all(), what
    err = float((got - want).abs().max() / want.abs().max().clamp(min=1e-30))
    assert err <= tolerance, (what, err, tolerance)


def _compare(got, want, dtype, time):
    f32 = _tolerance(torch.float32, time)
    _close(got[0], want[0], _tolerance(dtype, time), "y")
    _close(got[1], want[1], f32, "last")
    for name, g in want[2].items():
        _close(got[2][name], g, f32 if name in ("decay", "initial") else _tolerance(dtype, time), name)


SHAPES = [(1, 1, 1), (2, 15, 3), (1, 16, 64), (3, 17, 65), (1, 31, 129), (5, 64, 2), (2, 130, 130), (1, 300, 7),
          (3, 257, 200), (1, 1025, 33), (1, 4099, 18), (33, 130, 130), (70, 65, 3), (11, 200, 770)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("shape", SHAPES)
def test_matches_float64(shape, dtype):
    for reverse, resets, initial in ((False, 0.0, True), (True, 0.05, False)):
        t = _inputs(*shape, dtype, seed=sum(shape), resets=resets, initial=initial)
        print(shape, dtype, reverse, flush=True)
        _compare(_run(t, reverse), _reference(t, reverse), dtype, shape[1])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("channels", [64, 65, 66])
def test_strided_and_broadcast_inputs(dtype, channels):
    """Parts of one joint projection, time-major storage, a transposed tensor, a
    view that starts at an odd element, and an input that is the same at every step."""

    t = _inputs(2, 37, channels, dtype, seed=5, resets=0.1)
    want = _reference(t)
    joint = torch.cat([t["x"], t["recur"], t["input"]], -1).cuda().requires_grad_()
    x, recur, gate = joint.split(channels, -1)
    decay, initial = t["decay"].cuda(), t["initial"].cuda()
    y, last = gated_recurrence(x, recur, gate, decay, initial_state=initial, reset=t["reset"].cuda())
    (g,) = torch.autograd.grad((y, last), joint, (t["g_y"].cuda(), t["g_last"].cuda()))
    _close(y.detach(), want[0], _tolerance(dtype, 37), "joint y")
    for name, part in zip(("x", "recur", "input"), g.split(channels, -1)):
        _close(part, want[2][name], _tolerance(dtype, 37), "joint " + name)

    def time_major(v):
        return v.transpose(0, 1).contiguous().transpose(0, 1) if v.ndim == 3 else v

    def columns(v):
        return v.transpose(-1, -2).contiguous().transpose(-1, -2) if v.ndim == 3 else v

    def odd_start(v):
        return torch.nn.functional.pad(v, (1, 2))[..., 1:-2] if v.ndim == 3 else v

    for place in (time_major, columns, odd_start):
        _compare(_run(t, place=place), want, dtype, 37)

    # one gate for all steps: its gradient is the sum over them
    for name in ("recur", "input"):
        t[name] = t[name][:, :1].expand(-1, 37, -1)
    want = _reference(t)
    one = {k: t[k][:, :1].cuda().requires_grad_() for k in ("recur", "input")}
    y, _ = gated_recurrence(t["x"].cuda(), *(v.expand(-1, 37, -1) for v in one.values()), decay,
                            initial_state=initial, reset=t["reset"].cuda())
    _close(y.detach(), want[0], _tolerance(dtype, 37), "broadcast y")
    loss = (y.float() * t["g_y"].cuda().float()).sum()
    t["g_last"] = torch.zeros_like(t["g_last"])
    want = _reference(t)
    for name, g in zip(one, torch.autograd.grad(loss, list(one.values()))):
        # 37 rounded terms, and their sum rounded again
        limit = 38 * HALF_UNIT[dtype] + _tolerance(torch.float32, 37)
        _close(g, want[2][name].sum(1, keepdim=True), limit, "broadcast " + name)


def test_closed_and_open_gates():
    """Gates at the ends of their range: a closed gate (u = 0: the state stays as it
    is and the slope of s is infinite) and a state forgotten at once; finite gradients."""

    t = _inputs(2, 40, 64, torch.float32, seed=7)
    t["recur"][:, ::3] = -200.0
    t["recur"][:, 1::3] = -math.inf
    t["input"][:, ::5] = math.inf
    t["input"][:, 1::5] = -math.inf
    t["recur"][0, 2::3] = 60.0
    y, last, grads = _run(t)
    want = _reference(t, grads=False)
    _close(y, want[0], _tolerance(torch.float32, 40), "y")
    _close(last, want[1], _tolerance(torch.float32, 40), "last")
    for name, g in grads.items():
        assert torch.isfinite(g).all(), name
    # a closed gate passes no gradient to itself
    assert (grads["recur"][:, ::3] == 0).all() and (grads["recur"][:, 1::3] == 0).all()

    # decays so large that a_t is 0 in float32
    t = _inputs(1, 50, 64, torch.float32, seed=8)
    t["decay"][:32] = 40.0
    t["decay"][32:] = -60.0
    got, want = _run(t), _reference(t)
    _close(got[0], want[0], _tolerance(torch.float32, 50), "y")
    # (u is 1e-26 there: s is 1e-13, and so is what the input adds)
    _close(got[1], want[1], _tolerance(torch.float32, 50), "last")
    for name in ("x", "input", "initial"):
        _close(got[2][name], want[2][name], _tolerance(torch.float32, 50), name)


def test_decays_without_end():
    """Infinite decays and those near float32's ends: forgotten at once (a = 0) or
    kept for good (a = 1), a shut gate keeps either way; NaN stays in its channel."""

    for steps in (40, 200):
        t = _inputs(2, steps, 64, torch.float32, seed=28)
        t["recur"][:, 5:9] = -200.0
        t["recur"][:, 9] = -math.inf
        finite = dict(t, decay=torch.full((64,), 1e4))
        finite["decay"][32:] = -1e4
        want = _run(finite)
        _close(want[0], _reference(finite, grads=False)[0], _tolerance(torch.float32, steps), "y")
        for most in (math.inf, 3e38, 2.3e38, 1e20):
            t["decay"][:32], t["decay"][32:] = most, -most
            got = _run(t)
            # a, s and their slopes are the same for all of these
            assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1]), most
            for name in ("x", "input", "initial"):
                assert torch.equal(got[2][name], want[2][name]), (most, name)
            assert (got[2]["recur"] == 0).all() and torch.isfinite(got[2]["decay"]).all(), most
        t["decay"][3] = math.nan
        got = _run(t)
        others = torch.arange(64) != 3
        assert torch.isnan(got[0][..., 3]).all() and torch.equal(got[0][..., others], want[0][..., others])
    frame = [t[k][:, 5].cuda() for k in ("x", "recur", "input")]
    state = t["initial"].cuda()
    gated_recurrence_step(*frame, t["decay"].cuda(), state)
    assert torch.isnan(state[:, 3]).all() and torch.equal(state[:, others], t["initial"].cuda()[:, others])


def test_resets_drop_whatever_the_state_holds():
    """NaN and infinities before a reset, in the initial state too, do not reach
    the steps after it, nor the gradients of what comes after."""

    for dtype in (torch.float32, torch.bfloat16):
        t = _inputs(2, 300, 65, dtype, seed=9)
        t["reset"] = torch.zeros(2, 300, dtype=torch.bool)
        t["reset"][:, 0] = True
        t["reset"][0, 200] = True
        t["initial"][0] = math.nan
        t["initial"][1] = math.inf
        _compare(_run(t), _reference(t), dtype, 300)
        clean = _run(t)
        t["x"][0, 100:200] = math.nan
        t["x"][0, 150] = math.inf
        y, last, grads = _run(t)
        assert torch.equal(y[0, 200:], clean[0][0, 200:]) and torch.equal(last, clean[1])
        assert torch.equal(y[0, :100], clean[0][0, :100]) and torch.isnan(y[0, 100:200]).all()
        for name in ("x", "recur", "input"):
            assert torch.equal(grads[name][0, 200:], clean[2][name][0, 200:]), name
            assert torch.equal(grads[name][1], clean[2][name][1]), name


@pytest.mark.parametrize("reverse", [False, True])
@pytest.mark.parametrize("resets", [False, True])
def test_states_that_are_not_finite_stay_so(resets, reverse):
    """Over thousands of steps without a reset, whose factors' product is 0 in
    float32 (0.9^1024 is 1e-47), in both passes; and up to the reset where there is one."""

    def at(n):  # step n of the fold
        return time - 1 - n if reverse else n

    time = 4000
    t = _inputs(2, time, 66, torch.float32, seed=10)
    t["recur"].fill_(20.0)
    t["decay"].fill_(math.log(math.expm1(-math.log(0.9) / 8.0)))
    if resets:
        t["reset"] = torch.zeros(2, time, dtype=torch.bool)
        t["reset"][0, at(3000)] = True
    for bad in (math.nan, math.inf, -math.inf):
        t["initial"][0, :33] = bad
        t["x"][1, at(10), 33:] = bad
        y, last, _ = _run(t, reverse)
        y = y.flip(1) if reverse else y
        end = 3000 if resets else time
        assert not torch.isfinite(y[0, :end, :33]).any()
        assert not torch.isfinite(y[1, 10:, 33:]).any() and not torch.isfinite(last[1, 33:]).any()
        assert torch.isfinite(y[0, end:]).all() and torch.isfinite(last[0, :33]).all() == resets
        assert torch.isfinite(y[0, :, 33:]).all() and torch.isfinite(y[1, :10]).all() and torch.isfinite(y[1, :, :33]).all()

    # the gradient's carry, towards earlier steps
    t = dict(t, x=torch.randn(2, time, 66), initial=torch.randn(2, 66))
    t["g_last"][0, :33] = math.nan
    t["g_y"][1, at(3500), 33:] = math.inf
    _, _, grads = _run(t, reverse)
    g = grads["x"].flip(1) if reverse else grads["x"]
    assert not torch.isfinite(g[0, end if resets else 0:, :33]).any()
    assert not torch.isfinite(g[1, :3501, 33:]).any()
    assert not torch.isfinite(grads["initial"][1, 33:]).any()
    assert torch.isfinite(grads["initial"][0, :33]).all() == resets
    if resets:
        assert torch.isfinite(g[0, :end, :33]).all()
    assert torch.isfinite(g[1, 3501:]).all() and torch.isfinite(g[:, :, 33:][0]).all()


def test_every_step_reset_and_empty_sizes():
    t = _inputs(2, 35, 64, torch.float32, seed=11)
    t["reset"] = torch.ones(2, 35, dtype=torch.bool)
    got = _run(t)
    _compare(got, _reference(t), torch.float32, 1)
    assert (got[2]["initial"] == 0).all()

    for shape in ((0, 5, 4), (2, 0, 4), (2, 5, 0)):
        t = _inputs(*shape, torch.float32)
        y, last, grads = _run(t)
        assert y.shape == shape and last.shape == (shape[0], shape[2])
        assert torch.equal(last.cpu(), t["initial"]) or shape[1]
        if shape[1] == 0:
            assert torch.equal(grads["initial"].cpu(), t["g_last"])
        assert (grads["decay"] == 0).all()


def test_sequence_in_pieces_and_frame_by_frame():
    """Passing the last state on, in pieces and one frame at a time, gives the
    sequence's results; the state is updated in place."""

    for dtype in (torch.float32, torch.float16):
        t = _inputs(3, 50, 70, dtype, seed=13)
        x, recur, gate, decay = (t[k].cuda() for k in ("x", "recur", "input", "decay"))
        y, last = gated_recurrence(x, recur, gate, decay, initial_state=t["initial"].cuda())
        state, parts = t["initial"].cuda(), []
        for a, b in ((0, 1), (1, 33), (33, 50)):
            part, state = gated_recurrence(x[:, a:b], recur[:, a:b], gate[:, a:b], decay, initial_state=state)
            parts.append(part)
        want = _reference(t, grads=False)
        for got in (torch.cat(parts, 1), y):
            _close(got, want[0], _tolerance(dtype, 50), "y")
        _close(state, want[1], _tolerance(torch.float32, 50), "last")
        state = t["initial"].cuda()
        module = HipGatedRecurrence(70).cuda()
        module.decay.data.copy_(decay)
        for n in range(50):
            held = state.data_ptr()
            out = module.step(x[:, n], recur[:, n], gate[:, n], state)
            assert state.data_ptr() == held and not out.requires_grad
            _close(out, want[0][:, n], 2 * _tolerance(dtype, 50), f"frame {n}")
        _close(state, want[1], _tolerance(torch.float32, 50), "state")


def test_a_step_marks_its_state_as_changed():
    """What has saved the state for its backward raises there, as after torch's own
    updates in place; a state that requires a gradient is refused."""

    t = {k: v.cuda() for k, v in _inputs(2, 8, 16, torch.float32, seed=14).items() if v is not None}
    x, recur, gate, decay = t["x"].requires_grad_(), t["recur"], t["input"], t["decay"]
    frame = x[:, 0].detach(), recur[:, 0], gate[:, 0], decay
    _, last = gated_recurrence(x, recur, gate, decay)
    loss = last.square().sum()
    with pytest.raises(RuntimeError, match="require a gradient"):
        gated_recurrence_step(*frame, last)
    with pytest.raises(RuntimeError, match="require a gradient"):
        gated_recurrence_step(*frame, torch.zeros(2, 16, device="cuda", requires_grad=True))
    torch.autograd.grad(loss, x, retain_graph=True)
    gated_recurrence_step(*frame, last.detach())
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(loss, x)
    with torch.inference_mode():
        state = torch.zeros(2, 16, device="cuda")
        assert torch.isfinite(gated_recurrence_step(*frame, state)).all() and (state != 0).any()
    with torch.no_grad():
        gated_recurrence_step(*frame, torch.zeros(2, 16, device="cuda", requires_grad=True))


def test_gradient_against_differences():
    """The directional derivative of a weighted sum of the outputs, against its
    central difference: the step's cube (1e-2) and float32 results set 2e-3."""

    t = _inputs(2, 90, 40, torch.float32, seed=17, resets=0.05)
    _, _, grads = _run(t)
    g = torch.Generator().manual_seed(18)
    for name in NAMES:
        along = torch.randn(t[name].shape, generator=g)
        along = torch.sign(grads[name].cpu()) * along.abs()  # no cancellation between elements
        values = []
        for side in (1e-2, -1e-2):
            moved = {k: None if t[k] is None else t[k].cuda() for k in NAMES}
            moved[name] = moved[name] + side * along.cuda()
            y, last = gated_recurrence(moved["x"], moved["recur"], moved["input"], moved["decay"],
                                       initial_state=moved["initial"], reset=t["reset"].cuda())
            values.append(float((y.double().cpu() * t["g_y"].double()).sum()
                                + (last.double().cpu() * t["g_last"].double()).sum()))
        want = float((grads[name].double().cpu() * along.double()).sum())
        assert abs((values[0] - values[1]) / 2e-2 - want) <= 2e-3 * abs(want), (name, values, want)


def test_reproducible_and_on_another_stream():
    t = _inputs(4, 700, 96, torch.bfloat16, seed=19, resets=0.01)
    want = _run(t)
    side = torch.cuda.Stream()
    for _ in range(3):
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            got = _run(t)
        side.synchronize()
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
        for name, g in want[2].items():
            assert torch.equal(got[2][name], g), name


def test_only_the_gradients_that_are_asked_for():
    t = _inputs(2, 40, 33, torch.float32, seed=23)
    full = _run(t)[2]
    for name in NAMES:
        d = {k: t[k].cuda() for k in NAMES}
        d[name].requires_grad_()
        y, last = gated_recurrence(d["x"], d["recur"], d["input"], d["decay"], initial_state=d["initial"])
        (g,) = torch.autograd.grad((y, last), d[name], (t["g_y"].cuda(), t["g_last"].cuda()))
        assert torch.equal(g, full[name]), name
    # one output's gradient alone
    d = {k: t[k].cuda().requires_grad_() for k in NAMES}
    y, last = gated_recurrence(*(d[k] for k in NAMES[:4]), initial_state=d["initial"])
    grads = torch.autograd.grad(last, list(d.values()), t["g_last"].cuda())
    t["g_y"].zero_()
    for got, want in zip(grads, _run(t)[2].values()):
        assert torch.equal(got, want)
    # a second derivative is refused
    y, _ = gated_recurrence(*(d[k] for k in NAMES[:4]))
    (g,) = torch.autograd.grad(y.square().sum(), d["x"], create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable"):
        g.sum().backward()


def test_gradients_of_gradients_are_refused_whatever_the_upstream():
    """A penalty on a gradient next to another loss: refused where the gradient is a
    function of an input that wants one, also under a constant upstream; where it is
    not (y is linear in x and the initial state), its second derivative is 0."""

    t = _inputs(2, 20, 33, torch.float32, seed=25)
    #            of a gradient of                          by the inputs
    depends = {"x": {"recur", "input", "decay"}, "recur": set(NAMES), "input": {"x", "recur", "input", "decay"},
               "decay": set(NAMES), "initial": {"recur", "decay"}}
    for of in NAMES:
        for by in NAMES:
            d = {k: t[k].cuda() for k in NAMES}
            for name in (of, by):
                d[name].requires_grad_()
            y, last = gated_recurrence(*(d[k] for k in NAMES[:4]), initial_state=d["initial"])
            (g,) = torch.autograd.grad(y.sum() + last.sum(), d[of], create_graph=True)
            loss = g.square().sum() + sum(v.square().sum() for v in d.values())
            # (with `of` = `by` alone, what matters is whether the gradient depends on itself)
            if depends[of] & {of, by}:
                with pytest.raises(RuntimeError, match="once_differentiable"):
                    loss.backward()
            else:
                loss.backward()
                assert torch.equal(d[by].grad, 2 * d[by].detach()), (of, by)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float64])
def test_decays_of_other_types(dtype):
    """A module converted as a whole: the decay's value in float32, and its gradient
    rounded to its own type."""

    module = HipGatedRecurrence(48).cuda().to(dtype)
    assert module.decay.dtype == dtype
    t = _inputs(2, 40, 48, torch.bfloat16 if dtype == torch.float64 else dtype, seed=27)
    t["decay"] = module.decay.detach().float().cpu()
    want = _run(t)
    frames = [t[k].cuda() for k in ("x", "recur", "input")]
    y, last = module(*frames, initial_state=t["initial"].cuda())
    assert torch.equal(y, want[0]) and torch.equal(last, want[1])
    (g,) = torch.autograd.grad((y, last), module.decay, (t["g_y"].cuda(), t["g_last"].cuda()))
    assert g.dtype == dtype and torch.equal(g, want[2]["decay"].to(dtype))
    state = t["initial"].cuda()
    out = module.step(*(v[:, 0] for v in frames), state)
    assert torch.equal(out, gated_recurrence_step(*(v[:, 0] for v in frames), t["decay"].cuda(), t["initial"].cuda()))
    with pytest.raises(RuntimeError, match="decay"):
        gated_recurrence(*frames, torch.zeros(48, dtype=torch.int32, device="cuda"))


def test_forward_mode_is_refused():
    """A tangent on any input raises, whether gradients are recorded or not."""

    t = {k: v.cuda() for k, v in _inputs(2, 8, 16, torch.float32, seed=26).items() if v is not None}
    t["state"] = torch.zeros(2, 16, device="cuda")
    with forward_ad.dual_level():
        for name in (*NAMES, "state"):
            d = dict(t, **{name: forward_ad.make_dual(t[name], torch.ones_like(t[name]))})
            for recorded in (True, False):
                with torch.set_grad_enabled(recorded), pytest.raises(RuntimeError, match="jvp"):
                    if name == "state":
                        gated_recurrence_step(*(d[k][:, 0] for k in NAMES[:3]), d["decay"], d["state"])
                    else:
                        gated_recurrence(*(d[k] for k in NAMES[:4]), initial_state=d["initial"])
        # in a level, but without a tangent
        gated_recurrence(*(t[k] for k in NAMES[:4]))
    x = t["x"].requires_grad_()
    with forward_ad.dual_level(), pytest.raises(RuntimeError, match="jvp"):
        gated_recurrence(forward_ad.make_dual(x, torch.ones_like(x)), *(t[k] for k in NAMES[1:4]))


def test_refusals():
    t = {k: v.cuda() for k, v in _inputs(2, 8, 16, torch.float32).items() if v is not None}
    x, recur, gate, decay = t["x"], t["recur"], t["input"], t["decay"]
    with pytest.raises(RuntimeError, match="live on a GPU"):
        gated_recurrence(x.cpu(), recur, gate, decay)
    with pytest.raises(RuntimeError, match="live on a GPU"):
        gated_recurrence(x, recur, gate, decay.cpu())
    with pytest.raises(RuntimeError, match="float32, bfloat16 or float16"):
        gated_recurrence(x.double(), recur.double(), gate.double(), decay)
    with pytest.raises(RuntimeError, match="type of x"):
        gated_recurrence(x, recur.half(), gate, decay)
    with pytest.raises(RuntimeError, match="shape of x"):
        gated_recurrence(x, recur[:, :4], gate, decay)
    with pytest.raises(RuntimeError, match="batch, time, channels"):
        gated_recurrence(x[0], recur[0], gate[0], decay)
    with pytest.raises(RuntimeError, match="decay"):
        gated_recurrence(x, recur, gate, decay[:4])
    with pytest.raises(RuntimeError, match="initial_state"):
        gated_recurrence(x, recur, gate, decay, initial_state=t["initial"][:, :3])
    with pytest.raises(RuntimeError, match="reset"):
        gated_recurrence(x, recur, gate, decay, reset=torch.zeros(2, 8, device="cuda"))
    for rate in (0.0, -1.0, math.inf, math.nan):
        with pytest.raises(RuntimeError, match="rate has to be positive"):
            gated_recurrence(x, recur, gate, decay, rate=rate)
    with pytest.raises(RuntimeError, match="contiguous"):
        gated_recurrence_step(x[:, 0], recur[:, 0], gate[:, 0], decay, torch.zeros(16, 2, device="cuda").t())
    with pytest.raises(RuntimeError, match="state"):
        gated_recurrence_step(x[:, 0], recur[:, 0], gate[:, 0], decay, torch.zeros(2, 16, device="cuda").half())
    with pytest.raises(ValueError):
        HipGatedRecurrence(0)
    with pytest.raises(ValueError):
        HipGatedRecurrence(4, rate=0.0)
    with pytest.raises(ValueError):
        HipGatedRecurrence(4, fastest=0.99, slowest=0.9)
