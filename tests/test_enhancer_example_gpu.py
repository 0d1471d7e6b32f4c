"""The example enhancer: recurrence, norms and optimizer in one training on the loss."""

import importlib.util
from pathlib import Path

import pytest
import torch

pytestmark = pytest.mark.gpu

SOURCE = Path(__file__).resolve().parents[1] / "examples" / "train_enhancer.py"


@pytest.fixture(scope="module")
def example():
    spec = importlib.util.spec_from_file_location("train_enhancer", SOURCE)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


@pytest.mark.parametrize("bits", [32, 8])
def test_training_lowers_the_loss(example, bits):
    losses, net = example.train(steps=40, batch=4, state_bits=bits, say=lambda *_: None)
    assert all(torch.isfinite(torch.tensor(losses)))
    assert sum(losses[-5:]) < sum(losses[:5])
    assert all(torch.isfinite(p).all() for p in net.parameters())


def test_parameter_gradients_match_float64(example):
    """One step's gradients against the same network in plain float64 operations: 60
    frames through two blocks multiply the operators' 1e-5 by a few."""

    torch.manual_seed(3)
    net = example.Enhancer(width=48, blocks=2).cuda()
    g = torch.Generator().manual_seed(4)
    magnitudes = torch.rand(3, 60, example.BINS, generator=g)
    up = torch.randn(3, 60, example.BINS, generator=g)
    (net.gains(magnitudes.cuda()) * up.cuda()).sum().backward()

    params = {k: p.detach().double().cpu().requires_grad_() for k, p in net.named_parameters()}

    def linear(x, name):
        return x @ params[name + ".weight"].t() + params[name + ".bias"]

    def norm(x, w):
        return x / torch.sqrt(x.square().mean(-1, keepdim=True) + 1e-6) * w

    x = linear(torch.log(magnitudes.double() + 1e-4), "encode")
    n = norm(x, params["first"])
    for k in range(2):
        at = f"blocks.{k}."
        v, recur, gate, read = linear(n, at + "project").split(48, -1)
        u = 8.0 * torch.nn.functional.softplus(params[at + "recurrence.decay"]) * torch.sigmoid(recur)
        a, b = torch.exp(-u), torch.sqrt(-torch.expm1(-2 * u)) * torch.sigmoid(gate) * v
        h, ys = torch.zeros_like(b[:, 0]), []
        for t in range(60):
            h = a[:, t] * h + b[:, t]
            ys.append(h)
        branch = linear(torch.stack(ys, 1), at + "out")
        y = branch * torch.nn.functional.silu(linear(read, at + "out_gate"))
        x = x + params[at + "scale"] * norm(y, params[at + "weight"])
        n = norm(x, params[f"next.{k}"])
    (torch.sigmoid(linear(n, "decode")) * up.double()).sum().backward()
    for name, p in net.named_parameters():
        want = params[name].grad
        err = float((p.grad.double().cpu() - want).abs().max() / want.abs().max())
        assert err < 2e-4, (name, err)


def test_live_stream_matches_the_whole_clip(example):
    torch.manual_seed(5)
    net = example.Enhancer(width=64, blocks=3).cuda()
    magnitudes = torch.rand(2, 80, example.BINS, generator=torch.Generator().manual_seed(6)).cuda()
    with torch.no_grad():
        whole = net.gains(magnitudes)
    stream = example.Stream(net, 2)
    live = torch.stack([stream(magnitudes[:, t]) for t in range(80)], 1)
    # the same float32 operations but for the products' and sums' order
    assert float((live - whole).abs().max()) < 1e-4
