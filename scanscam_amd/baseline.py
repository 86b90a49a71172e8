"""
Tensor-level loop over time, for tensors that do not live on a GPU.

This is the package's counterpart of the reference's ``scanscam/baseline.py:8-40``
(the path ``scanscam/op.py:34-35, 54-55`` takes when no native kernel applies).
It is differentiable by ``torch.autograd``. GPU tensors never come here: they
go to the HIP kernels or raise.

Below it are the operators of a state space layer (``scanscam_amd.state_space``) in
the same manner: loops over time on tensors, differentiable by ``torch.autograd``,
in float64 where the inputs are and in float32 otherwise, rounded once at the end.
"""
from typing import List, Optional, Tuple

import torch
from torch.nn.functional import silu

from .decorator import preprocess_backward_scan_args, preprocess_scan_args


@preprocess_scan_args
def naive_linear_scan_forward(gate: torch.Tensor, value: torch.Tensor) -> torch.Tensor:
    T = gate.shape[1]
    state = torch.zeros_like(gate[:, 0])
    states: List[torch.Tensor] = []
    for t in range(T):
        state = state * gate[:, t] + value[:, t]
        states.append(state)
    if not states:
        return torch.empty_like(gate)
    return torch.stack(states, dim=1)


@preprocess_backward_scan_args
def naive_linear_scan_backward(
    gate: torch.Tensor, output: torch.Tensor, out_grad: torch.Tensor
) -> Tuple[torch.Tensor, torch.Tensor]:
    T = gate.shape[1]
    zero = torch.zeros_like(gate[:, 0])
    running = zero
    gate_grad: List[torch.Tensor] = [zero] * T
    value_grad: List[torch.Tensor] = [zero] * T
    for t in reversed(range(T)):
        running = running + out_grad[:, t]
        value_grad[t] = running
        gate_grad[t] = running * (output[:, t - 1] if t > 0 else zero)
        running = running * gate[:, t]
    if T == 0:
        return torch.empty_like(gate), torch.empty_like(gate)
    return torch.stack(gate_grad, dim=1), torch.stack(value_grad, dim=1)


def _wide(t: Optional[torch.Tensor]) -> Optional[torch.Tensor]:
    return t if t is None or t.dtype == torch.float64 else t.float()


def _sequences(x: torch.Tensor, offsets: Optional[torch.Tensor]) -> List[Tuple[int, int, int]]:
    """(batch element, first token, end) of every sequence."""
    if offsets is None:
        return [(b, 0, x.shape[1]) for b in range(x.shape[0])]
    ends = offsets.tolist()
    return [(0, a, b) for a, b in zip(ends[:-1], ends[1:])]


def _join(pieces: List[torch.Tensor], offsets: Optional[torch.Tensor], x: torch.Tensor) -> torch.Tensor:
    return (torch.stack(pieces) if offsets is None else torch.cat(pieces)[None]).to(x.dtype) if pieces else torch.empty_like(x)


def _rows_of(slots: Optional[torch.Tensor], rows: int, count: int) -> List[Tuple[int, int]]:
    """(token, row of the state) of the tokens that have one."""
    return [(i, s) for i, s in enumerate(range(rows) if slots is None else slots.tolist()) if 0 <= s < count]


def naive_selective_scan(x, dt, A, B, C, D=None, z=None, dt_bias=None, *, softplus=False, state=None, offsets=None, return_state=False):
    groups = 1 if B.dim() == 3 else B.shape[2]
    each = x.shape[2] // groups
    B, C = (_wide(v).reshape(*v.shape[:2], groups, v.shape[-1]).repeat_interleave(each, dim=2) for v in (B, C))
    wx, d, A, z = _wide(x), _wide(dt), _wide(A), _wide(z)
    if dt_bias is not None:
        d = d + _wide(dt_bias)
    if softplus:
        d = torch.logaddexp(d, torch.zeros_like(d))  # log(e^d + e^0), with a gradient of sigmoid(d) at zero too
    outs, states = [], []
    for s, (b, start, end) in enumerate(_sequences(x, offsets)):
        h = _wide(state[s]) if state is not None else torch.zeros_like(A)
        ys = []
        for t in range(start, end):
            h = torch.exp(d[b, t, :, None] * A) * h + (d[b, t] * wx[b, t])[:, None] * B[b, t]
            ys.append((C[b, t] * h).sum(-1))
        y = torch.stack(ys) if ys else wx[b, :0]
        if D is not None:
            y = y + _wide(D) * wx[b, start:end]
        if z is not None:
            y = y * silu(z[b, start:end])
        outs.append(y)
        states.append(h)
    y = _join(outs, offsets, x)
    return (y, torch.stack(states) if states else A.new_empty((0, *A.shape))) if return_state else y


def naive_selective_scan_step(state, x, dt, A, B, C, D=None, z=None, dt_bias=None, *, softplus=False, slots=None):
    y = torch.zeros_like(x)
    for i, s in _rows_of(slots, x.shape[0], state.shape[0]):
        row = [v if v is None else v[i][None, None] for v in (x, dt, B, C, z)]
        out, new = naive_selective_scan(row[0], row[1], A, row[2], row[3], D, row[4], dt_bias, softplus=softplus, state=state[s][None], return_state=True)
        y[i], state[s] = out[0, 0], new[0]
    return y


def naive_causal_conv(x, weight, bias=None, *, activation=None, state=None, offsets=None, return_state=False):
    K = weight.shape[1]
    w = _wide(weight)
    outs, states = [], []
    for s, (b, start, end) in enumerate(_sequences(x, offsets)):
        ahead = state[s] if state is not None else x.new_zeros((K - 1, x.shape[2]))
        rows = torch.cat((ahead, x[b, start:end]))
        wide, n = _wide(rows), end - start
        y = sum(w[:, k] * wide[k:k + n] for k in range(K))
        if bias is not None:
            y = y + _wide(bias)
        outs.append(silu(y) if activation == "silu" else y)
        states.append(rows[n:])
    y = _join(outs, offsets, x)
    return (y, torch.stack(states) if states else x.new_empty((0, K - 1, x.shape[2]))) if return_state else y


def naive_causal_conv_step(state, x, weight, bias=None, *, activation=None, slots=None):
    y = torch.zeros_like(x)
    for i, s in _rows_of(slots, x.shape[0], state.shape[0]):
        out, new = naive_causal_conv(x[i][None, None], weight, bias, activation=activation, state=state[s][None], return_state=True)
        y[i], state[s] = out[0, 0], new[0]
    return y


def naive_rms_norm(x, weight, residual=None, *, eps=1e-6, quant=None):
    total = x if residual is None else (_wide(x) + _wide(residual)).to(residual.dtype)
    wide = _wide(total)
    y = wide * torch.rsqrt((wide * wide).mean(-1, keepdim=True) + eps) * _wide(weight)
    if quant is None:
        y = y.to(x.dtype)
        return y if residual is None else (y, total)
    limit = 127.0 if quant == torch.int8 else 448.0
    most = y.abs().amax(-1) if y.shape[-1] else y.new_zeros(y.shape[:-1])
    scale = torch.where(most == 0, torch.ones_like(most), most / limit)
    q = (y / scale.unsqueeze(-1)).clamp(-limit, limit)
    q = q.round().to(quant) if quant == torch.int8 else q.to(quant)
    return (q, scale) if residual is None else (q, scale, total)
