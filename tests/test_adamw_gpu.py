"""AdamW over many tensors against the formula, moments in 32 and in 8 bits.

float32 updates carry about ten roundings (2^-24 each): 1e-6 of the largest
value after a step, and as much more per step.  8 bit codes follow from float32
values in a fixed order of operations, so a plain torch form in that order has
to give the same codes and scales bit for bit.
"""

import collections
import copy
import math

import pytest
import torch

from torch_pesq.hip_ops.adamw import HipAdamW

pytestmark = pytest.mark.gpu

HALF_UNIT = {torch.float32: 0.0, torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11}
SHAPES = [(1,), (3,), (255,), (256,), (257,), (0,), (17, 33), (1024,), (64, 257), (5, 3, 7), (1025,), (300, 301)]


def _params(dtype, seed=0, shapes=SHAPES):
    g = torch.Generator().manual_seed(seed)
    return [torch.nn.Parameter(torch.randn(s, generator=g).to(dtype).cuda()) for s in shapes]


def _grads(params, seed):
    g = torch.Generator().manual_seed(seed)
    out = []
    for p in params:
        size = 10 ** (4 * torch.rand((p.shape[0],) + (1,) * (p.ndim - 1), generator=g) - 3)
        out.append((torch.randn(p.shape, generator=g) * size).to(p.dtype).cuda())
    return out


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_32_bit_steps_match_float64(dtype):
    params = _params(dtype)
    opt = HipAdamW(params, lr=3e-3, betas=(0.8, 0.95), eps=1e-6, weight_decay=0.1)
    p64 = [p.detach().double() for p in params]
    m64, v64 = [torch.zeros_like(p) for p in p64], [torch.zeros_like(p) for p in p64]
    for step in range(1, 5):
        for k, (p, g) in enumerate(zip(params, _grads(params, step))):
            p.grad = g
            if dtype != torch.float32:
                p64[k] = p.detach().double()  # the stored value is what the step starts from
            g = g.double()
            m64[k] = 0.8 * m64[k] + 0.2 * g
            v64[k] = 0.95 * v64[k] + 0.05 * g * g
            hat = (m64[k] / (1 - 0.8**step)) / ((v64[k] / (1 - 0.95**step)).sqrt() + 1e-6)
            p64[k] = p64[k] * (1 - 3e-3 * 0.1) - 3e-3 * hat
        opt.step()
        for k, p in enumerate(params):
            if not p.numel():
                continue
            limit = HALF_UNIT[dtype] + 1e-6 * step
            assert float((p.detach().double() - p64[k]).abs().max() / p64[k].abs().max()) <= limit
            state = opt.state[p]
            assert state["step"] == step
            for got, want in ((state["exp_avg"], m64[k]), (state["exp_avg_sq"], v64[k])):
                assert got.shape == p.shape
                assert float((got.double() - want).abs().max() / want.abs().max()) <= 1e-6 * step


def _plain_codes(t, signed):
    blocks = torch.nn.functional.pad(t.reshape(-1), (0, -t.numel() % 256)).view(-1, 256)
    scale = blocks.abs().amax(1, keepdim=True)
    scale = torch.where(scale < 2.0**-100, torch.zeros_like(scale), scale)
    inverse = torch.where(scale > 0, 1.0 / scale, torch.zeros_like(scale))
    if signed:
        q = torch.round(torch.sqrt(blocks.abs() * inverse) * 127.0)
        q = torch.where(blocks < 0, -q, q).to(torch.int8)
    else:
        q = torch.round(torch.sqrt(torch.sqrt(blocks * inverse)) * 255.0)
        q = torch.where((blocks > 0) & (scale > 0), q.clamp(min=1.0), q).to(torch.uint8)
    return q.view(-1)[: t.numel()].view(t.shape), scale.view(-1)


def _plain_values(q, scale, signed):
    part = torch.nn.functional.pad(q.reshape(-1).float(), (0, -q.numel() % 256)).view(-1, 256)
    if signed:
        part = part / 127.0
        part = part.abs() * part
    else:
        part = part / 255.0
        part = part * part
        part = part * part
    return (part * scale.view(-1, 1)).view(-1)[: q.numel()].view(q.shape)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_8_bit_moments_match_the_plain_form_bit_for_bit(dtype):
    params = _params(dtype, seed=1)
    opt = HipAdamW(params, lr=2e-3, state_bits=8)
    plain = [p.detach().clone() for p in params]
    sizes = [None] * len(params)
    held = [(_plain_codes(torch.zeros(p.shape, device="cuda"), True),
             _plain_codes(torch.zeros(p.shape, device="cuda"), False)) for p in params]
    for step in range(1, 6):
        step_size, correction = 2e-3 / (1.0 - 0.9**step), 1.0 / math.sqrt(1.0 - 0.999**step)
        for k, (p, g) in enumerate(zip(params, _grads(params, 10 + step))):
            if step == 3:
                g.zero_()
            p.grad = g
            g = g.float()
            m = _plain_values(*held[k][0], True) * 0.9 + g * (1.0 - 0.9)
            v = _plain_values(*held[k][1], False) * 0.999 + (g * g) * (1.0 - 0.999)
            update = m / (torch.sqrt(v) * correction + 1e-8)
            plain[k] = (plain[k].float() * (1.0 - 2e-3 * 0.01) - update * step_size).to(dtype)
            sizes[k] = (update * step_size).double().abs()
            held[k] = (_plain_codes(m, True), _plain_codes(v, False))
        opt.step()
        flat = opt.moments()
        for k, p in enumerate(params):
            state = opt.state[p]
            # the step's quotient is four units off at most, and p rounded once
            off = (p.detach().double() - plain[k].double()).abs()
            assert (off <= 4 * 2.0**-23 * sizes[k] + (2.0**-23 + 2 * HALF_UNIT[dtype]) * plain[k].double().abs()).all(), (step, k)
            plain[k] = p.detach().clone()
            for name, (q, scale), signed in (("exp_avg", held[k][0], True), ("exp_avg_sq", held[k][1], False)):
                assert torch.equal(state[name], q), (step, k, name)
                assert torch.equal(state[name + "_scale"], scale), (step, k, name)
            for got, (q, scale), signed in zip(opt.moments(p), held[k], (True, False)):
                assert torch.equal(got, _plain_values(q, scale, signed)), (step, k)
            at = sum(-(-q.numel() // 256) * 256 for q in params[:k])
            assert torch.equal(flat[0][at : at + p.numel()], opt.moments(p)[0].view(-1))


def test_8_bit_codes_are_near_and_follow_32_bits():
    """Held values are within half a code's step of the moments (1.6 % of the value
    near the scale, absolute below), and training goes where 32 bits take it."""

    g = torch.Generator().manual_seed(3)
    target = torch.randn(40, 300, generator=g).cuda()
    last = {}
    for bits in (0, 32, 8):
        p = torch.nn.Parameter(torch.zeros(40, 300, device="cuda"))
        opt = (HipAdamW([p], lr=2e-2, weight_decay=0.0, state_bits=bits) if bits
               else torch.optim.AdamW([p], lr=2e-2, weight_decay=0.0))
        for _ in range(400):
            opt.zero_grad()
            ((p - target) ** 2).sum().backward()
            opt.step()
        last[bits] = float((p.detach() - target).abs().max())
    assert abs(last[32] - last[0]) <= 1e-3 * last[0] and last[8] <= 2 * last[0]

    p = torch.nn.Parameter(torch.zeros(512, device="cuda"))
    opt = HipAdamW([p], state_bits=8)
    p.grad = torch.logspace(-6, 0, 512).cuda()
    opt.step()
    m, v = (t.double() for t in opt.moments(p))
    grad = p.grad.double()
    for k in range(0, 512, 256):
        part = slice(k, k + 256)
        want_m, want_v = 0.1 * grad[part], 0.001 * grad[part] ** 2
        # half a step of the square root is sqrt(scale) / 254, of the fourth root scale^(1/4) / 510
        root = (m[part].sqrt() - want_m.sqrt()).abs().max() / want_m.max().sqrt()
        assert float(root) <= 1.001 / 254
        fourth = (v[part] ** 0.25 - want_v**0.25).abs() / want_v.max() ** 0.25
        assert float(fourth[v[part] > (1.5 / 255) ** 4 * want_v.max()].max()) <= 1.001 / 510
        assert (v[part] > 0).all()


def test_zero_tiny_and_non_finite_gradients():
    for bits in (32, 8):
        params = _params(torch.float32, seed=4, shapes=[(300,), (600,), (700,)])
        before = [p.detach().clone() for p in params]
        opt = HipAdamW(params, lr=1e-2, weight_decay=0.0, state_bits=bits)
        for p in params:
            p.grad = torch.zeros_like(p)
        params[1].grad.fill_(1e-32)
        params[2].grad[300] = math.nan
        params[2].grad[10] = math.inf
        opt.step()
        assert torch.equal(params[0], before[0])
        assert torch.isfinite(params[1]).all()
        # the two elements are lost, the others of this step are not
        bad = ~torch.isfinite(params[2].detach())
        assert bad.nonzero().view(-1).tolist() == [10, 300] and torch.equal(params[2][~bad], before[2][~bad])
        m, v = opt.moments(params[2])
        assert not torch.isfinite(m[10]) and torch.isnan(m[300]) and torch.isnan(v[300])
        if bits == 8:
            # their blocks' scales say so
            state = opt.state[params[2]]
            assert not torch.isfinite(state["exp_avg_scale"][:2]).any()
            assert torch.isfinite(state["exp_avg_scale"][2:]).all() and torch.isfinite(m[512:]).all()


def test_second_moment_beyond_float32():
    """A finite gradient whose square is infinite, then ordinary ones.  With 8 bits
    the block's scale is infinite, and its second moments are NaN from the next
    step on, like 0 times infinity in the plain form: so are its weights, and none
    takes a finite value from them.  With 32 bits that element alone stands still."""

    for bits in (32, 8):
        p = torch.nn.Parameter(torch.ones(600, device="cuda"))
        opt = HipAdamW([p], lr=1e-3, weight_decay=0.0, state_bits=bits)
        for step in range(3):
            p.grad = torch.full((600,), 1e-3, device="cuda")
            if step == 0:
                p.grad[5] = 2e19
            opt.step()
            if step == 0:
                assert p[5] == 1 and torch.isfinite(p).all()
        block = torch.zeros(600, dtype=torch.bool)
        if bits == 8:
            block[:256] = True
            assert torch.isnan(p.detach().cpu()[block]).all()
            assert torch.isinf(opt.state[p]["exp_avg_sq_scale"][0]) or torch.isnan(opt.state[p]["exp_avg_sq_scale"][0])
        else:
            block[5] = True
            assert p[5] == 1
        # the others take three full steps of the learning rate
        assert torch.allclose(p.detach().cpu()[~block], torch.tensor(1 - 3e-3), rtol=1e-5)


def test_without_eps():
    """eps = 0: no update where the moments are zero, a full one where the second
    moment is far below what its square can hold in float32."""

    for bits in (32, 8):
        p = torch.nn.Parameter(torch.ones(600, device="cuda"))
        opt = HipAdamW([p], lr=1e-2, eps=0.0, weight_decay=0.0, state_bits=bits)
        p.grad = torch.zeros_like(p)
        p.grad[300:] = 1e-3
        p.grad[400:] = 1e-25
        opt.step()
        assert (p[:300] == 1).all() and torch.isfinite(p).all()
        assert torch.allclose(p[300:400], torch.full((100,), 0.99, device="cuda"), rtol=1e-5)
        assert ((p[400:] > 0.98) & (p[400:] <= 1)).all()


def test_groups_missing_gradients_and_step_counts():
    """Groups with their own options, parameters without gradients (which keep their
    count), mixed types, non-contiguous gradients, many tensors."""

    for bits in (32, 8):
        shapes = [(k % 37 + 1, k % 11 + 1) for k in range(333)]
        params = _params(torch.float32, seed=5, shapes=shapes) + _params(torch.bfloat16, seed=6, shapes=shapes[:40])
        twins = [torch.nn.Parameter(p.detach().clone()) for p in params]
        opt = HipAdamW([{"params": params[::2], "lr": 1e-2}, {"params": params[1::2], "weight_decay": 0.2}],
                       lr=1e-3, state_bits=bits)
        for step in range(3):
            grads = _grads(params, 20 + step)
            for k, (p, g) in enumerate(zip(params, grads)):
                p.grad = None if (k + step) % 5 == 0 else g
                if k % 7 == 0 and p.grad is not None:
                    p.grad = g.t().contiguous().t()
            opt.step()
        for k, (p, twin) in enumerate(zip(params, twins)):
            # the same steps of this tensor alone
            alone = HipAdamW([twin], lr=1e-2 if k % 2 == 0 else 1e-3, weight_decay=0.2 if k % 2 else 1e-2,
                             state_bits=bits)
            if k % 29 == 0:
                for step in range(3):
                    if (k + step) % 5:
                        twin.grad = _grads(params, 20 + step)[k]
                        alone.step()
                assert torch.equal(p, twin), k
            assert opt.state[p]["step"] == sum((k + step) % 5 != 0 for step in range(3))


def test_views_and_unaligned_tensors():
    """Parameters and gradients that start anywhere in an allocation, and none of the
    elements next to them touched."""

    for dtype in (torch.float32, torch.bfloat16):
        for bits in (32, 8):
            flat = torch.full((5000,), 7.0, dtype=dtype, device="cuda")
            gflat = torch.full((5000,), 0.5, dtype=dtype, device="cuda")
            places = [(1, 300), (303, 1024), (1330, 515), (1900, 2048)]
            params, twins = [], []
            for a, n in places:
                p = torch.nn.Parameter(flat[a : a + n])
                p.grad = gflat[a + 3 : a + 3 + n]
                params.append(p)
                twin = torch.nn.Parameter(p.detach().clone())
                twin.grad = p.grad.clone()
                twins.append(twin)
            HipAdamW(params, state_bits=bits).step()
            HipAdamW(twins, state_bits=bits).step()
            inside = torch.zeros(5000, dtype=torch.bool)
            for (a, n), twin in zip(places, twins):
                assert torch.equal(flat[a : a + n], twin.detach())
                inside[a : a + n] = True
            assert (flat.cpu()[~inside] == 7.0).all() and (gflat == 0.5).all()


def test_state_round_trip_and_torch_s_state():
    params = _params(torch.float32, seed=7)
    for bits in (32, 8):
        mine = [torch.nn.Parameter(p.detach().clone()) for p in params]
        opt = HipAdamW(mine, lr=1e-2, state_bits=bits)
        for step in range(3):
            for p, g in zip(mine, _grads(mine, 30 + step)):
                p.grad = g
            opt.step()
        held = copy.deepcopy(opt.state_dict())
        other = [torch.nn.Parameter(p.detach().clone()) for p in mine]
        again = HipAdamW(other, lr=5e-1, state_bits=bits)
        again.load_state_dict(held)
        pickled = copy.deepcopy(again)
        for o, p, g in zip(other, mine, _grads(mine, 40)):
            o.grad, p.grad = g.clone(), g
        opt.step()
        again.step()
        for o, p in zip(other, mine):
            assert torch.equal(o, p) and again.state[o]["step"] == 4
        # the loaded tensors are copies
        assert held["state"][0]["step"] == 3
        for p, g in zip(pickled.param_groups[0]["params"], _grads(mine, 40)):
            p.grad = g
        pickled.step()
        for p, q in zip(pickled.param_groups[0]["params"], mine):
            assert torch.equal(p, q)
        with pytest.raises(ValueError, match="bits"):
            HipAdamW(other, state_bits=40 - bits).load_state_dict(held)
        with pytest.raises(ValueError, match="other parameter groups"):
            HipAdamW(other[:2], state_bits=bits).load_state_dict(held)

    # torch.optim.AdamW's state carries over, and its next step is ours
    a = [torch.nn.Parameter(p.detach().clone()) for p in params]
    theirs = torch.optim.AdamW(a, lr=1e-2)
    for p, g in zip(a, _grads(a, 50)):
        p.grad = g
    theirs.step()
    b = [torch.nn.Parameter(p.detach().clone()) for p in a]
    ours = HipAdamW(b, lr=1e-3)
    ours.load_state_dict(theirs.state_dict())
    for p, q, g in zip(a, b, _grads(a, 51)):
        p.grad, q.grad = g, g
    theirs.step()
    ours.step()
    for p, q in zip(a, b):
        assert torch.allclose(p, q, rtol=1e-5, atol=1e-6)
    assert ours.param_groups[0]["lr"] == 1e-2


@pytest.mark.parametrize("bits", [32, 8])
def test_a_load_that_fails_changes_nothing(bits):
    params = _params(torch.float32, seed=11, shapes=[(300,), (40, 40)])
    twins = [torch.nn.Parameter(p.detach().clone()) for p in params]
    opt, other = HipAdamW(params, state_bits=bits), HipAdamW(twins, state_bits=bits)

    def step(seed, *optimizers):
        for p, q, g in zip(params, twins, _grads(params, seed)):
            p.grad, q.grad = g, g.clone()
        for o in optimizers:
            o.step()

    step(80, opt, other)
    held = copy.deepcopy(opt.state_dict())
    bad = {
        "other shape": lambda s: s["state"][1].update(exp_avg=s["state"][1]["exp_avg"][:2].clone()),
        "other type": lambda s: s["state"][1].update(exp_avg_sq=s["state"][1]["exp_avg_sq"].double()),
        "other names": lambda s: s["state"][1].update(momentum_buffer=s["state"][1]["exp_avg"]),
        "no tensor": lambda s: s["state"][1].update(step="three"),
        "no state": lambda s: s["state"].update({1: None}),
        "no dictionary": lambda s: s.update(state=None),
    }
    for what, spoil in bad.items():
        spoiled = copy.deepcopy(held)
        for k in spoiled["state"]:
            spoiled["state"][k]["exp_avg"].fill_(3)
            spoiled["state"][k]["step"] = torch.tensor(77)
        spoil(spoiled)
        spoiled["param_groups"][0]["lr"] = 0.5
        with pytest.raises(Exception) as error:
            opt.load_state_dict(spoiled)
        assert isinstance(error.value, (ValueError, TypeError, RuntimeError, AttributeError)), (what, error.value)
        now = opt.state_dict()
        assert now["param_groups"] == held["param_groups"], what
        assert now["state"].keys() == held["state"].keys(), what
        for k, of in held["state"].items():
            assert all(torch.equal(torch.as_tensor(now["state"][k][name]).cpu(), t.cpu()) for name, t in of.items()), what
    step(81, opt, other)
    for p, q in zip(params, twins):
        assert torch.equal(p, q) and opt.state[p]["step"] == 2
        assert all(torch.equal(opt.state[p][name], other.state[q][name]) for name in opt.state[p])


@pytest.mark.parametrize("theirs,message", [
    (lambda p: torch.optim.AdamW(p, maximize=True), "maximize"),
    (lambda p: torch.optim.AdamW(p, amsgrad=True), "amsgrad"),
    (lambda p: torch.optim.Adam(p, weight_decay=0.1), "weight decay"),
    (lambda p: torch.optim.Adam(p), None),
])
def test_states_of_optimizers_that_step_otherwise(theirs, message):
    for stepped in (False, True):
        params = _params(torch.float32, seed=12, shapes=[(40, 40)])
        opt = theirs(params)
        if stepped:
            params[0].grad = _grads(params, 82)[0]
            opt.step()
        mine = HipAdamW(params, lr=0.25)
        if message is None:
            mine.load_state_dict(opt.state_dict())
            assert mine.param_groups[0]["lr"] == 1e-3 and mine.param_groups[0]["weight_decay"] == 0
            continue
        with pytest.raises(ValueError, match=message):
            mine.load_state_dict(opt.state_dict())
        assert mine.param_groups[0]["lr"] == 0.25 and not mine.state


@pytest.mark.parametrize("bits", [32, 8])
def test_load_runs_the_hooks_and_takes_every_option(bits):
    params = _params(torch.bfloat16, seed=13, shapes=[(300,), (40, 40)])
    opt = HipAdamW([{"params": params[:1], "name": "first"}, {"params": params[1:], "lr": 0.5}], state_bits=bits)
    for p, g in zip(params, _grads(params, 83)):
        p.grad = g
    opt.step()
    held = copy.deepcopy(opt.state_dict())
    held["param_groups"][1].update(max_lr=0.75, betas=[0.5, 0.25])

    other = HipAdamW([{"params": params[:1]}, {"params": params[1:]}], state_bits=bits)
    seen = []

    def before(optimizer, state_dict):
        seen.append(("before", len(optimizer.state)))
        # an older name of the moments
        state = {k: {n.replace("average", "exp_avg"): t for n, t in of.items()} for k, of in state_dict["state"].items()}
        return dict(state_dict, state=state)

    def after(optimizer):
        seen.append(("after", [int(optimizer.state[p]["step"]) for p in params]))

    other.register_load_state_dict_pre_hook(before)
    other.register_load_state_dict_post_hook(after)
    renamed = dict(held, state={k: {n.replace("exp_avg", "average"): t for n, t in of.items()}
                                for k, of in held["state"].items()})
    with pytest.raises(ValueError, match="bits"):
        other.load_state_dict(dict(renamed, param_groups=[dict(g, state_bits=40 - bits) for g in held["param_groups"]]))
    assert seen == [("before", 0)] and not other.state
    other.load_state_dict(renamed)
    assert seen == [("before", 0), ("before", 0), ("after", [1, 1])]
    assert other.param_groups[0]["name"] == "first" and other.param_groups[1]["max_lr"] == 0.75
    assert other.param_groups[1]["lr"] == 0.5 and tuple(other.param_groups[1]["betas"]) == (0.5, 0.25)
    for k, p in enumerate(params):
        assert all(torch.equal(other.state[p][n], torch.as_tensor(t)) for n, t in held["state"][k].items())
        assert other.state[p]["exp_avg"].dtype == (torch.float32 if bits == 32 else torch.int8)
    # back into torch's own, and from it
    if bits == 32:
        theirs = torch.optim.AdamW([{"params": params[:1]}, {"params": params[1:]}])
        theirs.load_state_dict(other.state_dict())
        other.load_state_dict(theirs.state_dict() | {"state": held["state"]})
        assert other.param_groups[1]["lr"] == 0.5 and other.state_bits == 32
    with pytest.raises(ValueError, match="learning rate"):
        other.load_state_dict(dict(renamed, param_groups=[dict(g, lr=-1.0) for g in held["param_groups"]]))


@pytest.mark.parametrize("bits", [32, 8])
def test_edits_of_state_and_groups_are_followed(bits):
    """A cleared or replaced state, tensors put into it, and parameters put into or taken
    out of a group count from the next step on, as in torch's optimizers."""

    params = _params(torch.float32, seed=14, shapes=[(300,), (40, 40), (257,)])

    def fresh(of):
        return [torch.nn.Parameter(p.detach().clone()) for p in of]

    def params_of(opt):
        return opt.param_groups[0]["params"]

    def step(opt, seed):
        ps = params_of(opt)
        for p, g in zip(ps, _grads(ps, seed)):
            p.grad = g
        opt.step()

    def same(a, b):
        for p, q in zip(params_of(a), params_of(b)):
            assert torch.equal(p, q)
            assert a.state[p].keys() == b.state[q].keys()
            assert all(torch.equal(a.state[p][n], b.state[q][n]) for n in a.state[p])
            assert all(torch.equal(x, y) for x, y in zip(a.moments(p), b.moments(q)))

    def clear(opt):
        opt.state.clear()

    def replace(opt):
        opt.state = collections.defaultdict(dict)

    def delete(opt):
        for p in params_of(opt):
            del opt.state[p]

    for forget in (clear, replace, delete):
        opt = HipAdamW(fresh(params), state_bits=bits)
        for seed in range(3):
            step(opt, 90 + seed)
        forget(opt)
        again = HipAdamW(fresh(params_of(opt)), state_bits=bits)
        for seed in range(2):
            step(opt, 95 + seed)
            step(again, 95 + seed)
            same(opt, again)
        assert len(opt.state_dict()["state"]) == 3

    # a tensor of the state, a count, one parameter's whole state
    for put in (lambda o, p: o.state[p].update(exp_avg=torch.zeros_like(o.state[p]["exp_avg"])),
                lambda o, p: o.state[p].update(step=40),
                lambda o, p: o.state.__setitem__(p, {})):
        opt = HipAdamW(fresh(params), state_bits=bits)
        step(opt, 100)
        put(opt, params_of(opt)[0])
        held = copy.deepcopy(opt.state_dict())
        again = HipAdamW(fresh(params_of(opt)), state_bits=bits)
        again.load_state_dict(held)
        step(opt, 101)
        step(again, 101)
        same(opt, again)

    # other parameters in the group
    opt = HipAdamW(fresh(params), state_bits=bits)
    step(opt, 110)
    gone = params_of(opt)[1]
    params_of(opt)[1] = torch.nn.Parameter(torch.ones(70, device="cuda"))
    before = gone.detach().clone()
    step(opt, 111)
    assert torch.equal(gone, before)
    assert [int(opt.state[p]["step"]) for p in params_of(opt)] == [2, 1, 2]
    opt.param_groups[0]["params"] = params_of(opt)[:1]
    step(opt, 112)
    assert int(opt.state[params_of(opt)[0]]["step"]) == 3
    # a tensor that does not fit is refused, and nothing has changed
    p = params_of(opt)[0]
    held, before = dict(opt.state[p]), p.detach().clone()
    opt.state[p]["exp_avg"] = torch.zeros(5, device="cuda")
    with pytest.raises(ValueError, match="exp_avg"):
        step(opt, 113)
    assert torch.equal(p, before)
    opt.state[p]["exp_avg"] = held["exp_avg"]
    step(opt, 113)
    assert int(opt.state[p]["step"]) == 4


def test_group_added_later_keeps_the_moments():
    params = _params(torch.float32, seed=8, shapes=[(300,), (40, 40)])
    for bits in (32, 8):
        opt = HipAdamW(params[:1], state_bits=bits)
        params[0].grad = _grads(params, 60)[0]
        opt.step()
        before = [t.clone() for t in opt.moments(params[0])]
        opt.add_param_group({"params": params[1:], "lr": 1e-2})
        for t, want in zip(opt.moments(params[0]), before):
            assert torch.equal(t, want)
        params[1].grad = _grads(params, 61)[1]
        opt.step()
        assert opt.state[params[0]]["step"] == 2 and opt.state[params[1]]["step"] == 1
        with pytest.raises(ValueError, match="not one of"):
            opt.moments(torch.nn.Parameter(torch.zeros(3)))


def test_closure_scheduler_version_and_streams():
    for bits in (32, 8):
        params = _params(torch.float32, seed=9, shapes=[(513,), (100, 70)])
        twins = [torch.nn.Parameter(p.detach().clone()) for p in params]
        opt, other = HipAdamW(params, state_bits=bits), HipAdamW(twins, state_bits=bits)
        schedule = torch.optim.lr_scheduler.StepLR(opt, 1, 0.5)
        side = torch.cuda.Stream()
        for step in range(3):
            for p, q, g in zip(params, twins, _grads(params, 70 + step)):
                p.grad, q.grad = g, g.clone()
            version = params[0]._version
            assert opt.step(lambda: 1.25) == 1.25
            assert params[0]._version > version
            schedule.step()
            other.param_groups[0]["lr"] = 1e-3 * 0.5**step
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):
                other.step()
            torch.cuda.current_stream().wait_stream(side)
        for p, q in zip(params, twins):
            assert torch.equal(p, q)


@pytest.mark.parametrize("bits", [8, 32])
def test_parameters_without_elements_alone(bits):
    params = _params(torch.float32, shapes=[(0,), (3, 0)])
    opt = HipAdamW(params, state_bits=bits)
    for p in params:
        p.grad = torch.zeros_like(p)
    opt.step()
    assert [int(opt.state[p]["step"]) for p in params] == [1, 1]
    assert [m.shape for m in opt.moments(params[1])] == [(3, 0), (3, 0)]


def test_refusals():
    p = torch.nn.Parameter(torch.zeros(4, 4, device="cuda"))
    for bad in ({"lr": -1.0}, {"lr": math.nan}, {"betas": (1.0, 0.9)}, {"betas": (0.9, -0.1)}, {"eps": -1e-8},
                {"weight_decay": -0.1}, {"state_bits": 16}):
        with pytest.raises(ValueError):
            HipAdamW([p], **bad)
    host = torch.nn.Parameter(torch.zeros(4))
    opt = HipAdamW([host])
    host.grad = torch.zeros(4)
    with pytest.raises(RuntimeError, match="live on a GPU"):
        opt.step()
    wide = torch.nn.Parameter(torch.zeros(4, device="cuda", dtype=torch.float64))
    wide.grad = torch.zeros_like(wide)
    with pytest.raises(RuntimeError, match="float32, bfloat16 or float16"):
        HipAdamW([wide]).step()
    strided = torch.nn.Parameter(torch.zeros(4, 6, device="cuda").t())
    strided.grad = torch.zeros(6, 4, device="cuda")
    with pytest.raises(RuntimeError, match="contiguous"):
        HipAdamW([strided]).step()
    p.grad = torch.zeros(4, 4, device="cuda").to_sparse()
    with pytest.raises(RuntimeError, match="dense"):
        HipAdamW([p]).step()
