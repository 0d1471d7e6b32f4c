"""A small recurrent speech enhancer trained on the PESQ loss, and run live.

The network maps the noisy signal's STFT magnitudes (frames of 512 samples, hop
256) to a gain per bin.  Its blocks are residual: a projection to the recurrence's
input, its two gates and an output gate, the gated recurrence over frames, a
projection back; ``residual_norm`` ends one block and starts the next.  Training
runs whole clips, with ``HipAdamW``; ``Stream`` runs the same network one frame at
a time, as a live enhancer does.

    python examples/train_enhancer.py --steps 200
"""

import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "triton-pesq_amd"))

from torch_pesq import PesqLossTriton  # noqa: E402
from torch_pesq.hip_ops.adamw import HipAdamW  # noqa: E402
from torch_pesq.hip_ops.norm import pre_norm, residual_norm  # noqa: E402
from torch_pesq.hip_ops.recurrence import HipGatedRecurrence  # noqa: E402

N_FFT, HOP = 512, 256
BINS = N_FFT // 2 + 1


class Block(torch.nn.Module):
    def __init__(self, width):
        super().__init__()
        self.project = torch.nn.Linear(width, 4 * width)
        self.recurrence = HipGatedRecurrence(width)
        self.out = torch.nn.Linear(width, width)
        self.out_gate = torch.nn.Linear(width, width)
        self.weight = torch.nn.Parameter(torch.ones(width))
        self.scale = torch.nn.Parameter(torch.full((width,), 0.2))

    def forward(self, n, state=None):
        """The branch and its gate from the normalised input, and the state after it.
        ``n`` is [batch, frames, width], or [batch, width] of one frame of a stream
        whose ``state`` is updated in place."""

        x, recur, gate, read = self.project(n).split(n.shape[-1], -1)
        if n.ndim == 2:
            y = self.recurrence.step(x, recur, gate, state)
        else:
            y, state = self.recurrence(x, recur, gate, initial_state=state)
        return self.out(y), self.out_gate(read), state


class Enhancer(torch.nn.Module):
    """Gains [..., bins] of STFT magnitudes [..., bins]."""

    def __init__(self, width=128, blocks=3):
        super().__init__()
        self.width = width
        self.encode = torch.nn.Linear(BINS, width)
        self.first = torch.nn.Parameter(torch.ones(width))
        self.blocks = torch.nn.ModuleList(Block(width) for _ in range(blocks))
        self.next = torch.nn.ParameterList(torch.nn.Parameter(torch.ones(width)) for _ in range(blocks))
        self.decode = torch.nn.Linear(width, BINS)

    def gains(self, magnitudes, states=None):
        x = self.encode(torch.log(magnitudes + 1e-4))
        n = pre_norm(x, self.first)
        for k, block in enumerate(self.blocks):
            branch, gate, _ = block(n, None if states is None else states[k])
            x, n = residual_norm(x, branch, block.weight, gate=gate, scale=block.scale, next_weight=self.next[k])
        return torch.sigmoid(self.decode(n))

    def forward(self, signal):
        """[batch, samples] -> [batch, samples]."""

        window = torch.hann_window(N_FFT, device=signal.device)
        spec = torch.stft(signal, N_FFT, HOP, window=window, return_complex=True)
        gains = self.gains(spec.abs().transpose(1, 2)).transpose(1, 2)
        return torch.istft(spec * gains, N_FFT, HOP, window=window, length=signal.shape[-1])


class Stream:
    """The gains of ``batch`` live streams, frame by frame."""

    def __init__(self, net, batch):
        self.net = net
        device = net.first.device
        self.states = [torch.zeros(batch, net.width, device=device) for _ in net.blocks]

    @torch.no_grad()
    def __call__(self, magnitudes):
        """[batch, bins] of the next frame -> [batch, bins]."""

        return self.net.gains(magnitudes, self.states)


def synthetic_speech(batch, samples, generator, device, rate=16000):
    """Harmonics of a gliding pitch in syllables: something PESQ can rate without data."""

    t = torch.arange(samples, device=device) / rate
    pitch = 100 + 120 * torch.rand(batch, 1, generator=generator, device=device)
    phase = 2 * torch.pi * pitch * (t + 0.004 * torch.sin(2 * torch.pi * 4 * t))
    signal = sum(torch.sin(k * phase) / k for k in range(1, 16))
    syllables = torch.rand(batch, samples // 4000 + 1, generator=generator, device=device) > 0.25
    signal = signal * syllables.float().repeat_interleave(4000, 1)[:, :samples] * torch.sin(2 * torch.pi * 2 * t) ** 2
    return 0.05 * signal / signal.square().mean(1, keepdim=True).sqrt().clamp(min=1e-3)


def train(steps=200, batch=8, seconds=2.0, state_bits=32, lr=2e-3, seed=0, say=print):
    """Losses of the steps, and the trained network."""

    torch.manual_seed(seed)
    generator = torch.Generator(device="cuda").manual_seed(seed)
    net = Enhancer().cuda()
    pesq = PesqLossTriton(1.0, sample_rate=16000).cuda()
    opt = HipAdamW(net.parameters(), lr=lr, state_bits=state_bits)
    losses = []
    for step in range(steps):
        clean = synthetic_speech(batch, int(seconds * 16000), generator, "cuda")
        noisy = clean + 0.02 * torch.randn(clean.shape, generator=generator, device="cuda")
        loss = pesq(clean, net(noisy)).mean()
        opt.zero_grad()
        loss.backward()
        opt.step()
        losses.append(loss.detach())
        if step % 20 == 0 or step == steps - 1:
            say(f"step {step:4d}  loss {float(losses[-1]):.4f}")
    return torch.stack(losses).tolist(), net


def main():
    parser = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    parser.add_argument("--steps", type=int, default=200)
    parser.add_argument("--batch", type=int, default=8)
    parser.add_argument("--state-bits", type=int, default=32, choices=(32, 8))
    args = parser.parse_args()
    _, net = train(args.steps, args.batch, state_bits=args.state_bits)
    # the last clip again, as a live stream
    generator = torch.Generator(device="cuda").manual_seed(1)
    clean = synthetic_speech(1, 32000, generator, "cuda")
    spec = torch.stft(clean, N_FFT, HOP, window=torch.hann_window(N_FFT, device="cuda"), return_complex=True).abs()
    with torch.no_grad():
        whole = net.gains(spec.transpose(1, 2))
    stream = Stream(net, 1)
    live = torch.stack([stream(frame) for frame in spec.unbind(-1)], 1)
    print(f"live and whole clip differ by {float((live - whole).abs().max()):.2e} in gain")


if __name__ == "__main__":
    main()
