"""The network operators beyond 32 bit offsets, in HIP graphs and on streams at once.

Each result is compared with the same call on small, contiguous, eager tensors,
bit for bit: neither strides nor how the call is made may change it.
"""

import copy

import pytest
import torch

from torch_pesq.hip_ops.adamw import HipAdamW
from torch_pesq.hip_ops.norm import residual_norm
from torch_pesq.hip_ops.recurrence import gated_recurrence

pytestmark = pytest.mark.gpu

FAR = 2**31 + 2**20  # elements


def _recurrence_inputs(shape, dtype=torch.bfloat16, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    t = [torch.randn(shape, generator=g, device="cuda").to(dtype) for _ in range(3)]
    decay = -4.0 - 4.0 * torch.rand(shape[-1], generator=g, device="cuda")
    up = torch.randn(shape, generator=g, device="cuda").to(dtype)
    return t, decay, up


def _recurrence_step(t, decay, up):
    leaves = [v.detach().requires_grad_() for v in t]
    y, last = gated_recurrence(*leaves, decay)
    return [y.detach(), last.detach(), *torch.autograd.grad(y, leaves, up)]


def _same(got, want):
    for a, b in zip(got, want):
        assert torch.equal(a, b)


def test_recurrence_rows_far_apart():
    t, decay, up = _recurrence_inputs((3, 300, 70))
    want = _recurrence_step(t, decay, up)
    far = torch.zeros(2 * FAR + 10**6, dtype=torch.bfloat16, device="cuda")
    spread = far.as_strided(t[0].shape, (FAR, 70, 1))
    spread.copy_(t[0])
    _same(_recurrence_step([spread, t[1], t[2]], decay, up), want)
    up_far = far.as_strided(up.shape, (FAR, 80, 1), 500_000)
    up_far.copy_(up)
    _same(_recurrence_step([t[0], t[1], t[2]], decay, up_far), want)
    # steps as far apart as the operator takes them, and further: copied
    for stride in (2**26 - 2, 2**26 + 2):
        steps = far.as_strided((1, 60, 70), (0, stride, 1))
        part = [v[:1, :60].contiguous() for v in t]
        steps.copy_(part[1])
        _same(_recurrence_step([part[0], steps, part[2]], decay, up[:1, :60].contiguous()),
              _recurrence_step(part, decay, up[:1, :60].contiguous()))


def test_recurrence_float32_steps_far_apart():
    """Below 2^27 bytes apart as they are, from there on copied; both directions."""

    t, decay, up = _recurrence_inputs((1, 60, 70), torch.float32)
    far = torch.zeros(60 * (2**25 + 2), device="cuda")
    for stride in (2**25 - 2, 2**25 + 2):
        steps = far.as_strided((1, 60, 70), (0, stride, 1))
        steps.copy_(t[1])
        _same(_recurrence_step([t[0], steps, t[2]], decay, up), _recurrence_step(t, decay, up))
        for reverse in (False, True):
            _same([gated_recurrence(t[0], steps, t[2], decay, reverse=reverse)[0]],
                  [gated_recurrence(*t, decay, reverse=reverse)[0]])
        steps.copy_(up)
        _same(_recurrence_step(t, decay, steps), _recurrence_step(t, decay, up))


def test_recurrence_larger_than_32_bits():
    """More than 2^31 elements of y: the last rows against the same rows alone."""

    shape = (34, 64000, 1024)
    x = torch.full((1, 1, 1), 0.5, dtype=torch.bfloat16, device="cuda").expand(shape)
    tail, decay, _ = _recurrence_inputs((1, 64000, 1024), seed=3)
    gate = tail[1].expand(shape)
    y, last = gated_recurrence(x, gate, gate, decay)
    want, want_last = gated_recurrence(x[:1], tail[1], tail[1], decay)
    for row in (0, 32, 33):
        assert torch.equal(y[row], want[0]) and torch.equal(last[row], want_last[0])


def test_norm_rows_far_apart():
    g = torch.Generator(device="cuda").manual_seed(5)
    x, branch, gate = (torch.randn(5, 264, generator=g, device="cuda").bfloat16() for _ in range(3))
    w = torch.rand(264, generator=g, device="cuda") + 0.5

    def step(x, branch, gate):
        leaves = [v.detach().requires_grad_() for v in (x, branch, gate)]
        out = residual_norm(leaves[0], leaves[1], w, gate=leaves[2], scale=w, next_weight=w)
        return [*(o.detach() for o in out), *torch.autograd.grad(out, leaves, (branch, gate))]

    far = torch.zeros(3 * (FAR // 2) + 4 * FAR // 4, dtype=torch.bfloat16, device="cuda")
    spread = far.as_strided(x.shape, (FAR // 2, 1))
    spread.copy_(branch)
    _same(step(x, spread, gate), step(x, branch, gate))


@pytest.mark.parametrize("bits", [32, 8])
def test_adamw_tensor_of_more_than_2_31_elements(bits):
    count = 2**31 + 777
    p = torch.nn.Parameter(torch.full((count,), 0.5, dtype=torch.bfloat16, device="cuda"))
    p.grad = torch.zeros(count, dtype=torch.bfloat16, device="cuda")
    g = torch.Generator(device="cuda").manual_seed(6)
    end = torch.randn(3000, generator=g, device="cuda").bfloat16()
    p.grad[-3000:] = end
    small = torch.nn.Parameter(torch.full((3000,), 0.5, dtype=torch.bfloat16, device="cuda"))
    small.grad = end.clone()
    for q in (p, small):
        HipAdamW([q], lr=1e-1, state_bits=bits).step()
    assert torch.equal(p.detach()[-3000:], small.detach())
    assert (p.detach()[:-3000] == p.detach()[0]).all()


def test_forward_in_a_graph():
    """Captured once, replayed with new inputs between eager calls."""

    shape = (3, 700, 96)
    t, decay, _ = _recurrence_inputs(shape, seed=7)
    w = torch.rand(96, device="cuda") + 0.5

    def call():
        y, last = gated_recurrence(*t, decay)
        x, n = residual_norm(t[0], y, w, gate=t[1], next_weight=w)
        return [y, last, x, n]

    with torch.no_grad():
        call()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = call()
        for seed in range(8, 13):
            fresh, _, _ = _recurrence_inputs(shape, seed=seed)
            for v, f in zip(t, fresh):
                v.copy_(f)
            graph.replay()
            torch.cuda.synchronize()
            _same(out, call())


def test_optimizer_step_in_a_graph():
    """A captured step repeats its own step's corrections: the same as an eager one
    from the same count."""

    for bits in (32, 8):
        p, q = (torch.nn.Parameter(torch.linspace(-1, 1, 5000, device="cuda")) for _ in range(2))
        p.grad, q.grad = (torch.linspace(1, -1, 5000, device="cuda") for _ in range(2))
        captured, eager = HipAdamW([p], state_bits=bits), HipAdamW([q], state_bits=bits)
        captured.moments()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            captured.step()
        graph.replay()
        eager.step()
        torch.cuda.synchronize()
        assert torch.equal(p, q)
        _same(captured.moments(), eager.moments())


@pytest.mark.parametrize("bits", [32, 8])
def test_replays_of_a_captured_step_count(bits):
    """Every replay is a step of its own: moments and counts as after as many eager
    steps, and weights but for the corrections, which the GPU computes (one unit of
    float32 in two factors of the update, 2^-22 of it a step).  Eager steps between
    the replays count on, of other tensors too."""

    lr, shapes = 1e-2, [(300,), (0,), (40, 40), (1025,)] + [(k % 7 + 1, 9) for k in range(120)]

    def make():
        g = torch.Generator().manual_seed(30)
        params = [torch.nn.Parameter(torch.randn(s, generator=g).to(torch.bfloat16 if k % 5 == 4 else torch.float32).cuda())
                  for k, s in enumerate(shapes)]
        for p in params:
            p.grad = torch.zeros_like(p)
        return params, HipAdamW([{"params": params[:2]}, {"params": params[2:], "weight_decay": 0.0}], lr=lr, state_bits=bits)

    def fill(params, seed):
        g = torch.Generator(device="cuda").manual_seed(seed)
        for p in params:
            if p.grad is not None:
                p.grad.copy_(torch.randn(p.shape, generator=g, device="cuda"))

    (a, captured), (b, eager) = make(), make()
    steps = 0

    def check():
        torch.cuda.synchronize()
        _same(captured.moments(), eager.moments())
        for p, q in zip(a, b):
            assert int(captured.state[p]["step"]) == int(eager.state[q]["step"])
            unit = 2.0**-8 if p.dtype == torch.bfloat16 else 2.0**-23
            off = (p.detach().double() - q.detach().double()).abs()
            # an update is below 10 lr here; a weight is rounded once a step on either side
            assert (off <= steps * (2.0**-22 * 10 * lr + unit * (q.detach().double().abs() + 10 * lr))).all()

    for seed in range(2):
        fill(a, seed), fill(b, seed)
        captured.step(), eager.step()
        steps += 1
    check()
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        captured.step()
    check()
    for seed in range(2, 9):
        fill(a, seed), fill(b, seed)
        left = [(p, p.grad) for p in (a[2], b[2], a[7], b[7])]
        if seed in (4, 7):
            # an eager step, without two of the tensors
            for p, _ in left:
                p.grad = None
            captured.step()
        else:
            graph.replay()
        eager.step()
        for p, grad in left:
            p.grad = grad
        steps += 1
        check()
    # the counts in a state are those of what was enqueued before
    graph.replay()
    eager.step()
    steps += 1
    held = captured.state_dict()
    assert [int(of["step"]) for of in held["state"].values()] == [int(of["step"]) for of in eager.state_dict()["state"].values()]
    check()
    # a load reaches the graph
    held = copy.deepcopy(held)
    for _ in range(3):
        graph.replay()
    for p, q in zip(a, b):
        p.data.copy_(q.data)
    captured.load_state_dict(held)
    for seed in range(20, 23):
        fill(a, seed), fill(b, seed)
        graph.replay()
        eager.step()
        steps += 1
        check()
    captured.state.clear()
    assert captured.moments()[0].abs().max() == 0
    again = HipAdamW([{"params": b[:2]}, {"params": b[2:], "weight_decay": 0.0}], lr=lr, state_bits=bits)
    eager = again
    for p, q in zip(a, b):
        p.data.copy_(q.data)
    for seed in range(30, 32):
        fill(a, seed), fill(b, seed)
        graph.replay()
        eager.step()
        steps += 1
        check()
    # a copy counts by itself
    other = copy.deepcopy(captured)
    for p, q in zip((p for g in other.param_groups for p in g["params"]), b):
        p.grad = q.grad.clone()
    other.step()
    eager.step()
    assert [int(of["step"]) for of in other.state.values()] == [3] * len(shapes)
    _same(other.moments(), eager.moments())


def test_counts_outlive_their_optimizer():
    """Replays that are still to run when the optimizer goes count in memory that no
    other pinned tensor gets."""

    p = torch.nn.Parameter(torch.ones(2**24, device="cuda"))
    p.grad = torch.ones_like(p)
    opt = HipAdamW([p])
    opt.moments()
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        opt.step()
    for _ in range(200):
        graph.replay()
    del opt
    others = [torch.zeros(1, dtype=torch.int64, pin_memory=True) for _ in range(20)]
    torch.cuda.synchronize()
    assert all(int(t) == 0 for t in others)


def test_what_a_graph_cannot_hold():
    for bits in (32, 8):
        p = torch.nn.Parameter(torch.ones(300, device="cuda"))
        p.grad = torch.ones_like(p)
        opt = HipAdamW([p], state_bits=bits)
        torch.cuda.synchronize()
        with pytest.raises(RuntimeError, match="first step"):
            with torch.cuda.graph(torch.cuda.CUDAGraph()):
                opt.step()
        opt.step()
        torch.cuda.synchronize()
        assert int(opt.state[p]["step"]) == 1 and (p < 1).all()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            opt.step()
        opt.add_param_group({"params": [torch.nn.Parameter(torch.ones(4, device="cuda"))]})
        with pytest.raises(RuntimeError, match="stay as they are"):
            opt.step()
        del opt.param_groups[1]
        opt.step()
        torch.cuda.synchronize()
        assert int(opt.state[p]["step"]) == 2


def test_streams_at_once():
    """Two streams' recurrences of many chunks at the same time: each waits for its
    own pairs only."""

    cases = [_recurrence_inputs((2, 9000, 130), seed=20), _recurrence_inputs((40, 1500, 96), seed=21)]
    want = [_recurrence_step(*c) for c in cases]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    got = [None, None]
    for _ in range(5):
        for k, (c, s) in enumerate(zip(cases, streams)):
            with torch.cuda.stream(s):
                got[k] = _recurrence_step(*c)
    torch.cuda.synchronize()
    for a, b in zip(got, want):
        _same(a, b)
