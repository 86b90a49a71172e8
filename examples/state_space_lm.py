"""
A small state space language model on this package's operators: trained on a synthetic task, then asked to go on from
packed prompts of different lengths, token by token.

    python examples/state_space_lm.py [--device cuda|cpu] [--dtype bfloat16] [--channels 128] [--layers 2] [--steps 100]

A layer is  norm (with the residual's addition) -> projection to x and z -> short causal convolution -> projection to dt, B
and C -> selective scan, gated by z -> projection back.  Training and prompts go through ``rms_norm``, ``causal_conv`` and
``selective_scan``; a generated token through ``causal_conv_step`` and ``selective_scan_step``, which update the states of the
sequences in place. With ``eight`` set a layer's first projection takes its norm's output in 8 bits.

The task: after a first token the sequence repeats with a period of three, so that what comes next has to be kept in the states.
"""
import argparse
import math
import os
import sys

import torch
from torch import nn
from torch.nn import functional as F

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
from scanscam_amd import causal_conv, causal_conv_step, rms_norm, selective_scan, selective_scan_step  # noqa: E402


class Layer(nn.Module):
    def __init__(self, channels: int, states: int = 16, taps: int = 4):
        super().__init__()
        inner, rank = 2 * channels, max(1, channels // 16)
        self.inner, self.states, self.taps, self.rank = inner, states, taps, rank
        self.norm = nn.Parameter(torch.ones(channels))
        self.into = nn.Linear(channels, 2 * inner, bias=False)
        self.conv = nn.Parameter(torch.randn(inner, taps) / math.sqrt(taps))
        self.conv_bias = nn.Parameter(torch.zeros(inner))
        self.select = nn.Linear(inner, rank + 2 * states, bias=False)
        self.dt = nn.Linear(rank, inner, bias=False)
        steps = torch.exp(torch.rand(inner) * math.log(100.0) + math.log(1e-3))  # 0.001 to 0.1
        self.dt_bias = nn.Parameter(torch.log(torch.expm1(steps)))
        self.A_log = nn.Parameter(torch.log(torch.arange(1.0, states + 1)).repeat(inner, 1))
        self.D = nn.Parameter(torch.ones(inner))
        self.out = nn.Linear(inner, channels, bias=False)

    def new_states(self, sequences: int, like: torch.Tensor):
        """The inputs that the convolution keeps and the scan's states, of ``sequences`` sequences."""
        return (torch.zeros(sequences, self.taps - 1, self.inner, dtype=like.dtype, device=like.device),
                torch.zeros(sequences, self.inner, self.states, device=like.device))

    def _project(self, x, residual, eight):
        """x and z of the normalised sum, and the sum."""
        if eight is None:
            y, residual = rms_norm(x, self.norm, residual)
            return self.into(y), residual
        q, scale, residual = rms_norm(x, self.norm, residual, quant=eight)
        return self.into(q.to(x.dtype)) * scale.unsqueeze(-1).to(x.dtype), residual

    def _selection(self, x):
        dt, B, C = self.select(x).split((self.rank, self.states, self.states), dim=-1)
        return self.dt(dt), B, C

    def forward(self, x, residual, offsets=None, keep=False, eight=None):
        """Whole sequences, [batch, T, channels], or packed ones; with ``keep`` their states after the last tokens as well."""
        xz, residual = self._project(x, residual, eight)
        x, z = xz.chunk(2, dim=-1)
        conv = causal_conv(x, self.conv, self.conv_bias, activation="silu", offsets=offsets, return_state=keep)
        x, kept = conv if keep else (conv, None)
        dt, B, C = self._selection(x)
        y = selective_scan(x, dt, -torch.exp(self.A_log), B, C, self.D, z, self.dt_bias, softplus=True, offsets=offsets, return_state=keep)
        y, state = y if keep else (y, None)
        return self.out(y), residual, (kept, state)

    def step(self, x, residual, states, slots=None, eight=None):
        """One token of each of several sequences, [rows, channels]."""
        kept, state = states
        xz, residual = self._project(x, residual, eight)
        x, z = xz.chunk(2, dim=-1)
        x = causal_conv_step(kept, x, self.conv, self.conv_bias, activation="silu", slots=slots)
        dt, B, C = self._selection(x)
        y = selective_scan_step(state, x, dt, -torch.exp(self.A_log), B, C, self.D, z, self.dt_bias, softplus=True, slots=slots)
        return self.out(y), residual


class Model(nn.Module):
    def __init__(self, vocabulary: int = 32, channels: int = 128, layers: int = 2):
        super().__init__()
        self.embedding = nn.Embedding(vocabulary, channels)
        nn.init.normal_(self.embedding.weight, std=channels ** -0.5)
        self.layers = nn.ModuleList(Layer(channels) for _ in range(layers))
        self.norm = nn.Parameter(torch.ones(channels))

    def _logits(self, x, residual):
        y, _ = rms_norm(x, self.norm, residual)
        return F.linear(y, self.embedding.weight)

    def forward(self, tokens, offsets=None, keep=False, eight=None):
        """Logits of [batch, T] tokens, and with ``keep`` the states of all layers."""
        x = self.embedding(tokens)
        residual, states = torch.zeros_like(x, dtype=torch.float32), []
        for layer in self.layers:
            x, residual, kept = layer(x, residual, offsets, keep, eight)
            states.append(kept)
        return (self._logits(x, residual), states) if keep else self._logits(x, residual)

    def step(self, tokens, states, slots=None, eight=None):
        """Logits of one token of each of several sequences, [rows]."""
        x = self.embedding(tokens)
        residual = torch.zeros_like(x, dtype=torch.float32)
        for layer, kept in zip(self.layers, states):
            x, residual = layer.step(x, residual, kept, slots, eight)
        return self._logits(x, residual)


def sequences(batch, T, vocabulary, generator, device):
    """[batch, T] tokens that repeat with a period of three after the first."""
    three = torch.randint(1, vocabulary, (batch, 3), generator=generator)
    return three.repeat(1, T // 3 + 1)[:, :T].to(device)


def train(model, steps, device, batch=16, T=96, vocabulary=32, seed=0):
    """The loss of every step."""
    generator = torch.Generator().manual_seed(seed)
    optimizer = torch.optim.AdamW(model.parameters(), lr=3e-3)
    losses = []
    for _ in range(steps):
        tokens = sequences(batch, T + 1, vocabulary, generator, device)
        logits = model(tokens[:, :-1])
        loss = F.cross_entropy(logits.flatten(0, 1).float(), tokens[:, 1:].flatten())
        optimizer.zero_grad()
        loss.backward()
        optimizer.step()
        losses.append(loss.item())
    return losses


@torch.no_grad()
def generate(model, prompts, count, eight=None):
    """``count`` tokens after each of the prompts (lists of tokens, of any lengths), which go through the model as one packed batch."""
    if any(len(p) == 0 for p in prompts):
        raise ValueError("an empty prompt has no token to go on from")
    if not prompts or count < 1:
        return [[] for _ in prompts]
    device = model.norm.device
    offsets = torch.tensor([0] + [len(p) for p in prompts], dtype=torch.int32).cumsum(0, dtype=torch.int32).to(device)
    packed = torch.tensor([t for p in prompts for t in p], device=device).unsqueeze(0)
    logits, states = model(packed, offsets=offsets, keep=True, eight=eight)
    token = logits[0, offsets[1:].long() - 1].argmax(-1)
    out = [token]
    for _ in range(count - 1):
        token = model.step(token, states, eight=eight).argmax(-1)
        out.append(token)
    return torch.stack(out, 1).tolist()


def main(argv=None):
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--device", default="cuda" if torch.cuda.is_available() else "cpu")
    ap.add_argument("--dtype", default="float32", choices=("float32", "bfloat16", "float16"))
    ap.add_argument("--channels", type=int, default=128)
    ap.add_argument("--layers", type=int, default=2)
    ap.add_argument("--steps", type=int, default=100)
    a = ap.parse_args(argv)
    torch.manual_seed(0)
    model = Model(channels=a.channels, layers=a.layers).to(a.device)
    losses = train(model, a.steps, a.device)
    print(f"loss {losses[0]:.3f} -> {losses[-1]:.3f} after {a.steps} steps")
    model = model.to(getattr(torch, a.dtype))
    prompts = [[5, 9, 2, 5, 9, 2, 5], [7, 1, 30] * 9 + [7, 1], [11, 12, 13, 11]]
    for eight in (None, torch.float8_e4m3fn):
        out = generate(model, prompts, 9, eight)
        right = sum(o == [p[(len(p) + i) % 3] for i in range(9)] for p, o in zip(prompts, out))
        print(f"{'8-bit projections' if eight else a.dtype}: {right} of {len(prompts)} prompts continued as they should be: {out}")
    return losses, out


if __name__ == "__main__":
    main()
