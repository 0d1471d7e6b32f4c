"""The residual norm against the formula in float64.

A float32 result has some ten roundings in its chain (2^-24 each) and sums over
the row whose error grows as the logarithm of its length at most: 2e-6 of the
row's largest value, and 1e-5 for sums over rows that cancel in part; 16 bit
results half a unit of their type more.  The gradient through a norm is what is
left of its argument without the part along the row: with few channels that can
be little of it, so these 2e-6 are of the terms before the difference.
"""

import math

import pytest
import torch
import torch.autograd.forward_ad as forward_ad

from torch_pesq.hip_ops.norm import pre_norm, residual_norm

pytestmark = pytest.mark.gpu

HALF_UNIT = {torch.float32: 0.0, torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11}
NAMES = ("x", "branch", "gate", "weight", "scale", "next_weight")
TYPES = [(torch.float32, torch.float32), (torch.bfloat16, torch.bfloat16), (torch.float16, torch.float16),
         (torch.float32, torch.bfloat16), (torch.float32, torch.float16)]


def _inputs(shape, stream, dtype, seed=0, without=()):
    g = torch.Generator().manual_seed(seed)
    level = 10 ** (2 * torch.rand(shape[:-1] + (1,), generator=g) - 1)
    t = {"x": (torch.randn(shape, generator=g) * level).to(stream),
         "branch": (torch.randn(shape, generator=g) * level).to(dtype),
         "gate": torch.randn(shape, generator=g).to(dtype)}
    for name, mean in (("weight", 1.0), ("scale", 0.3), ("next_weight", 1.0)):
        t[name] = mean + 0.1 * torch.randn(shape[-1], generator=g)
    for name in without:
        t[name] = None
    up = {"x_out": torch.randn(shape, generator=g).to(stream), "n": torch.randn(shape, generator=g).to(dtype)}
    return t, up


def _reference(t, up, eps=1e-6):
    d = {k: None if v is None else v.double().requires_grad_() for k, v in t.items()}
    y = d["branch"]
    if d["gate"] is not None:
        y = y * torch.nn.functional.silu(d["gate"])
    z = y / torch.sqrt(y.square().mean(-1, keepdim=True) + eps) * d["weight"]
    x = d["x"] + (z if d["scale"] is None else d["scale"] * z)
    out = {"x_out": x}
    if d["next_weight"] is not None:
        out["n"] = x / torch.sqrt(x.square().mean(-1, keepdim=True) + eps) * d["next_weight"]
    names = [k for k in NAMES if d[k] is not None]
    grads = torch.autograd.grad(list(out.values()), [d[k] for k in names], [up[k].double() for k in out])
    # the largest term of each row's gradients
    with torch.no_grad():
        top = {"x": up["x_out"].double().abs()}
        if "n" in out:
            top["x"] = top["x"] + (up["n"] * d["next_weight"]).abs() / torch.sqrt(x.square().mean(-1, keepdim=True) + eps)
        of_y = top["x"] * d["weight"].abs() / torch.sqrt(y.square().mean(-1, keepdim=True) + eps)
        if d["scale"] is not None:
            of_y = of_y * d["scale"].abs()
        top["branch"] = of_y
        if d["gate"] is not None:
            sig = torch.sigmoid(d["gate"])
            top["branch"] = of_y * (d["gate"] * sig).abs()
            top["gate"] = of_y * (d["branch"] * sig * (1 + d["gate"] * (1 - sig))).abs()
    return {k: v.detach() for k, v in out.items()}, dict(zip(names, grads)), top


def _run(t, up, eps=1e-6, place=lambda v: v):
    d = {k: None if v is None else place(v.cuda()).detach().requires_grad_() for k, v in t.items()}
    out = residual_norm(d["x"], d["branch"], d["weight"], gate=d["gate"], scale=d["scale"],
                        next_weight=d["next_weight"], eps=eps)
    out = {"x_out": out} if d["next_weight"] is None else dict(zip(("x_out", "n"), out))
    names = [k for k in NAMES if d[k] is not None]
    grads = torch.autograd.grad(list(out.values()), [d[k] for k in names], [up[k].cuda() for k in out])
    return {k: v.detach() for k, v in out.items()}, dict(zip(names, grads))


def _check(got, want, t, up):
    for name, value in want[0].items():
        assert got[0][name].dtype == up[name].dtype
        _close(got[0][name], value, HALF_UNIT[up[name].dtype] + 2e-6, name)
    for name, value in want[1].items():
        assert got[1][name].dtype == t[name].dtype
        wide = name in NAMES[3:]
        _close(got[1][name], value, HALF_UNIT[t[name].dtype] + (1e-5 if wide else 2e-6), "d" + name, want[2].get(name))


def _close(got, want, tolerance, what, top=None):
    """Row by row, since rows are of very different size: against the largest of
    ``top``, or of the row itself."""

    assert got.shape == want.shape, what
    got = got.double().cpu()
    assert torch.isfinite(got).all(), what
    if not want.numel():
        return
    err = (got - want).abs().reshape(-1, want.shape[-1]).amax(1)
    top = torch.maximum(want.abs(), want.abs() if top is None else top)
    err = float((err / top.reshape(-1, want.shape[-1]).amax(1).clamp(min=1e-30)).max())
    assert err <= tolerance, (what, err, tolerance)


SHAPES = [(1, 1), (3, 2), (1, 7), (5, 63), (4, 64), (130, 65), (3, 256), (37, 257), (9, 512), (600, 40), (2, 1000),
          (70, 1024), (3, 2049), (5, 4096), (2, 8191), (3, 8192)]


@pytest.mark.parametrize("stream,dtype", TYPES)
@pytest.mark.parametrize("shape", SHAPES)
def test_matches_float64(shape, stream, dtype):
    print(shape, stream, dtype, flush=True)
    t, up = _inputs(shape, stream, dtype, seed=sum(shape))
    if shape[-1] == 1:
        # the norm of one channel is its sign: gradients through it are pure rounding
        got, want = _run(t, up), _reference(t, up)
        for name in want[0]:
            _close(got[0][name], want[0][name], HALF_UNIT[up[name].dtype] + 2e-6, name)
        return
    _check(_run(t, up), _reference(t, up), t, up)


@pytest.mark.parametrize("without", [("gate",), ("scale",), ("next_weight",), ("gate", "scale"),
                                     ("gate", "next_weight"), ("gate", "scale", "next_weight")])
@pytest.mark.parametrize("stream,dtype", TYPES[::2] + TYPES[3:4])
def test_without_some_operands(without, stream, dtype):
    for shape in ((11, 300), (2, 5, 256), (33, 2056)):
        t, up = _inputs(shape, stream, dtype, seed=3, without=without)
        _check(_run(t, up), _reference(t, up), t, up)


@pytest.mark.parametrize("shape,dtype,result", [
    ((7, 257), torch.float32, None), ((7, 264), torch.bfloat16, None), ((3, 5, 2000), torch.float32, torch.bfloat16),
    ((1, 5000), torch.float16, None), ((400, 33), torch.float32, torch.float16),
])
def test_pre_norm(shape, dtype, result):
    t, up = _inputs(shape, dtype, result or dtype, seed=5)
    x, w = t["x"].double().requires_grad_(), t["weight"].double().requires_grad_()
    want = x / torch.sqrt(x.square().mean(-1, keepdim=True) + 1e-5) * w
    want_g = torch.autograd.grad(want, (x, w), up["n"].double())
    x, w = t["x"].cuda().requires_grad_(), t["weight"].cuda().requires_grad_()
    n = pre_norm(x, w, eps=1e-5, dtype=result)
    assert n.dtype == (result or dtype)
    g = torch.autograd.grad(n, (x, w), up["n"].cuda())
    _close(n.detach(), want.detach(), HALF_UNIT[n.dtype] + 2e-6, "n")
    _close(g[0], want_g[0], HALF_UNIT[dtype] + 2e-6, "dx")
    _close(g[1], want_g[1], 1e-5, "dw")


@pytest.mark.parametrize("channels", [64, 257, 520])
def test_strided_rows_and_batch_shapes(channels):
    """Halves of a joint projection, columns cut out of wider rows at an odd start,
    transposed storage, a broadcast gate, three-dimensional inputs."""

    for stream, dtype in ((torch.float32, torch.float32), (torch.bfloat16, torch.bfloat16)):
        t, up = _inputs((6, 5, channels), stream, dtype, seed=channels)
        want = _reference(t, up)
        for place in (lambda v: torch.cat([v, v], -1)[..., : v.shape[-1]] if v.ndim > 1 else v,
                      lambda v: torch.nn.functional.pad(v, (1, 2))[..., 1:-2],
                      lambda v: v.transpose(0, 1).contiguous().transpose(0, 1) if v.ndim > 1 else v,
                      lambda v: v.transpose(-1, -2).contiguous().transpose(-1, -2) if v.ndim > 1 else v):
            _check(_run(t, up, place=place), want, t, up)
        one = t["gate"][:1, :1].cuda().requires_grad_()
        t["gate"] = t["gate"][:1, :1].expand(6, 5, -1)
        want = _reference(t, up)
        x, n = residual_norm(t["x"].cuda(), t["branch"].cuda(), t["weight"].cuda(), gate=one.expand(6, 5, -1),
                             scale=t["scale"].cuda(), next_weight=t["next_weight"].cuda())
        _close(x.detach(), want[0]["x_out"], HALF_UNIT[stream] + 2e-6, "x_out")
        (g,) = torch.autograd.grad((x, n), one, (up["x_out"].cuda(), up["n"].cuda()))
        # thirty rounded terms of very different size, their sum rounded again
        sums = want[1]["gate"].abs().sum((0, 1)).max()
        err = (g.double().cpu()[0, 0] - want[1]["gate"].sum((0, 1))).abs().max()
        assert err <= (2 * HALF_UNIT[dtype] + 4e-6) * sums


def test_rows_of_zeros_and_of_the_type_s_ends():
    """Silent rows: eps alone under the root; finite gradients.  Values whose squares
    pass float32's range: the norm is 0 there and the row stays as it was."""

    t, up = _inputs((8, 96), torch.float32, torch.float32, seed=9)
    t["branch"][0] = 0
    t["gate"][1] = 0
    t["x"][2] = 0
    t["branch"][2] = 0
    t["x"][3] = 0
    t["branch"][4] *= 1e-30
    t["gate"][5] = 100.0
    t["gate"][6] = -100.0
    got, want = _run(t, up), _reference(t, up)
    for name, value in want[0].items():
        _close(got[0][name], value, 2e-6, name)
    for name, value in want[1].items():
        _close(got[1][name], value, 1e-5, "d" + name, want[2].get(name))
    t["gate"][:, ::2] = -1e30
    t["gate"][:, 1::2] = 1e4
    got = _run(t, up)
    for value in (*got[0].values(), *got[1].values()):
        assert torch.isfinite(value).all()


def test_nan_and_infinite_rows_stay_in_their_rows():
    t, up = _inputs((6, 320), torch.float32, torch.bfloat16, seed=10)
    clean = _run(t, up)
    t["x"][2, 5] = math.nan
    t["branch"][4, 7] = math.inf
    got = _run(t, up)
    rows = [0, 1, 3, 5]
    for name, value in got[0].items():
        assert torch.equal(value[rows], clean[0][name][rows]), name
        assert not torch.isfinite(value[2]).all() and not torch.isfinite(value[4]).all()
    for name in ("x", "branch", "gate"):
        assert torch.equal(got[1][name][rows], clean[1][name][rows]), name


def test_gradient_against_differences():
    """Central differences of a weighted sum of the outputs along each gradient's
    signs: the step's cube and float32 results set 2e-3."""

    t, up = _inputs((12, 100), torch.float32, torch.float32, seed=12)
    for name in ("x", "branch"):
        t[name] = t[name] / t[name].square().mean(-1, keepdim=True).sqrt()
    _, grads = _run(t, up)
    g = torch.Generator().manual_seed(13)
    for name in NAMES:
        along = torch.sign(grads[name].cpu()) * torch.randn(t[name].shape, generator=g).abs()
        values = []
        for side in (1e-2, -1e-2):
            d = {k: v.cuda() for k, v in t.items()}
            d[name] = d[name] + side * along.cuda()
            x, n = residual_norm(d["x"], d["branch"], d["weight"], gate=d["gate"], scale=d["scale"],
                                 next_weight=d["next_weight"])
            values.append(float((x.double().cpu() * up["x_out"].double()).sum()
                                + (n.double().cpu() * up["n"].double()).sum()))
        want = float((grads[name].double().cpu() * along.double()).sum())
        assert abs((values[0] - values[1]) / 2e-2 - want) <= 2e-3 * abs(want), (name, values, want)


def test_many_rows_reproducible_and_on_another_stream():
    t, up = _inputs((5000, 136), torch.bfloat16, torch.bfloat16, seed=14)
    want = _run(t, up)
    _check(want, _reference(t, up), t, up)
    side = torch.cuda.Stream()
    for _ in range(3):
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            got = _run(t, up)
        side.synchronize()
        for part, other in zip(got, want):
            for name, value in part.items():
                assert torch.equal(value, other[name]), name


def test_only_the_gradients_that_are_asked_for():
    t, up = _inputs((9, 130), torch.float32, torch.float32, seed=15)
    full = _run(t, up)[1]
    for name in NAMES:
        d = {k: v.cuda() for k, v in t.items()}
        d[name].requires_grad_()
        out = residual_norm(d["x"], d["branch"], d["weight"], gate=d["gate"], scale=d["scale"],
                            next_weight=d["next_weight"])
        (g,) = torch.autograd.grad(out, d[name], (up["x_out"].cuda(), up["n"].cuda()))
        assert torch.equal(g, full[name]), name
    for alone, other in ((0, "n"), (1, "x_out")):
        zero = dict(up, **{other: torch.zeros_like(up[other])})
        want = _run(t, zero)[1]
        d = {k: v.cuda().requires_grad_() for k, v in t.items()}
        out = residual_norm(d["x"], d["branch"], d["weight"], gate=d["gate"], scale=d["scale"],
                            next_weight=d["next_weight"])
        grads = torch.autograd.grad(out[alone], list(d.values()), zero[("x_out", "n")[alone]].cuda())
        for name, g in zip(d, grads):
            assert torch.allclose(g, want[name], rtol=1e-6, atol=0), name
    # weights of the branch's type
    d = {k: v.cuda().bfloat16().requires_grad_() for k, v in t.items()}
    out = residual_norm(d["x"], d["branch"], d["weight"], gate=d["gate"], scale=d["scale"],
                        next_weight=d["next_weight"])
    for g in torch.autograd.grad(out, list(d.values()), [v.cuda().bfloat16() for v in up.values()]):
        assert g.dtype == torch.bfloat16 and torch.isfinite(g).all()
    y = residual_norm(d["x"], d["branch"], d["weight"])
    (g,) = torch.autograd.grad(y.square().sum(), d["x"], create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable"):
        g.sum().backward()


def test_gradients_of_gradients_are_refused_whatever_the_upstream():
    """A penalty on a gradient next to another loss: refused where the gradient is a
    function of an input that wants one, also under a constant upstream; where it is
    not (x_out is linear in x, the weight and the scale), its second derivative is 0."""

    t, _ = _inputs((9, 130), torch.float32, torch.float32, seed=16)
    everything = set(NAMES)
    #                    of a gradient of                   by the inputs
    depends = {"x_out": {"x": set(), "branch": {"branch", "gate", "weight", "scale"},
                         "gate": {"branch", "gate", "weight", "scale"}, "weight": {"branch", "gate", "scale"},
                         "scale": {"branch", "gate", "weight"}, "next_weight": set()},
               "n": {**{k: everything for k in NAMES[:5]}, "next_weight": everything - {"next_weight"}}}
    for which, output in enumerate(depends):
        for of in NAMES:
            for by in NAMES:
                if output == "x_out" and of == "next_weight":
                    continue  # not connected
                d = {k: v.cuda() for k, v in t.items()}
                for name in (of, by):
                    d[name].requires_grad_()
                out = residual_norm(d["x"], d["branch"], d["weight"], gate=d["gate"], scale=d["scale"],
                                    next_weight=d["next_weight"])[which]
                (g,) = torch.autograd.grad(out.sum(), d[of], create_graph=True)
                loss = g.square().sum() + sum(v.square().sum() for v in d.values())
                if depends[output][of] & {of, by}:
                    with pytest.raises(RuntimeError, match="once_differentiable"):
                        loss.backward()
                else:
                    loss.backward()
                    assert torch.equal(d[by].grad, 2 * d[by].detach()), (output, of, by)
    x, w = t["x"].cuda().requires_grad_(), t["weight"].cuda()
    (g,) = torch.autograd.grad(pre_norm(x, w).sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable"):
        (x.sum() + g.square().sum()).backward()


def test_forward_mode_is_refused():
    """A tangent on any input raises, whether gradients are recorded or not; weights
    that are converted first among them."""

    t, _ = _inputs((4, 32), torch.float32, torch.float32, seed=17)
    t = {k: v.cuda() for k, v in t.items()}
    t["weight"] = t["weight"].half()
    with forward_ad.dual_level():
        for name in NAMES:
            d = dict(t, **{name: forward_ad.make_dual(t[name], torch.ones_like(t[name]))})
            for recorded in (True, False):
                with torch.set_grad_enabled(recorded), pytest.raises(RuntimeError, match="jvp"):
                    residual_norm(d["x"], d["branch"], d["weight"], gate=d["gate"], scale=d["scale"],
                                  next_weight=d["next_weight"])
        with pytest.raises(RuntimeError, match="jvp"):
            pre_norm(forward_ad.make_dual(t["x"], torch.ones_like(t["x"])), t["weight"])
        # in a level, but without a tangent
        residual_norm(t["x"], t["branch"], t["weight"])


def test_no_rows():
    t, up = _inputs((0, 40), torch.float32, torch.float32)
    got = _run(t, up)
    assert got[0]["x_out"].shape == (0, 40) and got[0]["n"].shape == (0, 40)
    for name in NAMES[3:]:
        assert (got[1][name] == 0).all()


def test_refusals():
    t, _ = _inputs((4, 32), torch.float32, torch.float32)
    d = {k: v.cuda() for k, v in t.items()}
    with pytest.raises(RuntimeError, match="live on a GPU"):
        residual_norm(t["x"], d["branch"], d["weight"])
    with pytest.raises(RuntimeError, match="live on a GPU"):
        residual_norm(d["x"], t["branch"], d["weight"])
    with pytest.raises(RuntimeError, match="live on a GPU"):
        pre_norm(d["x"], t["weight"])
    with pytest.raises(RuntimeError, match="needs a branch"):
        residual_norm(d["x"], None, d["weight"])
    with pytest.raises(RuntimeError, match="shape of x"):
        residual_norm(d["x"], d["branch"][:2], d["weight"])
    with pytest.raises(RuntimeError, match="type of the branch"):
        residual_norm(d["x"], d["branch"], d["weight"], gate=d["gate"].half())
    with pytest.raises(RuntimeError, match="has to be float32 or"):
        residual_norm(d["x"].half(), d["branch"].bfloat16(), d["weight"])
    with pytest.raises(RuntimeError, match="float32, bfloat16 or float16"):
        pre_norm(d["x"].double(), d["weight"])
    with pytest.raises(RuntimeError, match="float32, bfloat16 or float16"):
        pre_norm(d["x"], d["weight"], dtype=torch.float64)
    with pytest.raises(RuntimeError, match="channels"):
        residual_norm(d["x"], d["branch"], d["weight"][:3])
    with pytest.raises(RuntimeError, match="eps"):
        residual_norm(d["x"], d["branch"], d["weight"], eps=-1.0)
    wide = torch.zeros(1, 8193, device="cuda")
    with pytest.raises(RuntimeError, match="1 to 8192 channels"):
        pre_norm(wide, wide[0])
