"""
The operators of a linear attention layer in a language model: attention with a decay for each head, whose state is a matrix where the
selective scan's is a vector, over whole sequences with gradients and for single tokens, and the norm of its heads with their gate.

Tensors, types, packed sequences, single tokens' slots and recorded calls are as in ``scanscam_amd.state_space``: activations tokens-first
(``[batch, T, heads, channels of a head]``) in float32, bfloat16 or float16, states in float32, GPU tensors on the kernels of
``libscanscam_hip.so`` (C ABI in ``include/scanscam_attention.h``), CPU tensors on the loops of ``scanscam_amd.baseline``. None of this has a
counterpart in the reference, whose one operator is the scan.
"""
import ctypes
import operator
from typing import Optional, Tuple, Union

import torch

from . import baseline, hip, state_space
from .state_space import (_ACTIVATIONS, _MOST_CHANNELS, _TYPES, _Param, _Tokens, _bytes, _check_activation, _check_devices, _check_in_place, _check_offsets,
                          _check_saved, _check_shape, _check_sizes, _check_slots, _check_types, _dense, _eager, _f32, _has_tangent, _i32, _i64,
                          _meta, _near, _needs_node, _p, _param, _ptr, _raise, _rows, _size, _stream, _tokens, _traced_through, _unit, _wants_grad)

_MOST_HEAD, _MOST_GROUP = 256, 8192


class _Attend(ctypes.Structure):
    _fields_ = ([(n, _i64) for n in ("batch", "T", "sequences", "heads", "groups", "K", "V")] + [("offsets", _p)] +
                [(n, _i32) for n in ("offsets64", "dtype", "decay_dtype", "decay_fixed")] + [("scale", _f32), ("parts", _i32)] +
                [(n, _Tokens) for n in ("q", "k", "v", "y", "decay")] + [(n, _p) for n in ("state_in", "state_out", "saved")] +
                [(n, _Tokens) for n in ("gy", "gq", "gk", "gv")] + [(n, _p) for n in ("gdecay", "gstate_out", "gstate_in", "workspace")] +
                [("workspace_bytes", _size)])


class _AttendStep(ctypes.Structure):
    _fields_ = ([(n, _i64) for n in ("rows", "heads", "groups", "K", "V", "slots")] + [("slot", _p)] +
                [(n, _i32) for n in ("slot64", "dtype", "decay_dtype")] + [("scale", _f32)] +
                [(n, _Tokens) for n in ("q", "k", "v", "y", "decay")] + [("state", _p)])


class _GroupNorm(ctypes.Structure):
    _fields_ = ([(n, _i64) for n in ("rows", "channels", "groups", "x_stride", "z_stride")] + [("x", _p), ("z", _p)] +
                [("weight", _Param), ("bias", _Param), ("y", _p), ("eps", _f32)] + [(n, _i32) for n in ("dtype", "activation", "unused")] +
                [(n, _p) for n in ("gy", "gx", "gz", "gweight", "gbias", "workspace")] + [("workspace_bytes", _size)])


_entry_points = None
# Parts of time that a sequence is shared out in; 0: the library chooses (the tests force others).
_parts = 0


def _lib():
    """The library with these operators' entry points bound; raises where they are missing."""
    global _entry_points
    if _entry_points is None:
        lib = hip.lib()
        for name, args in (("attend_fwd", _Attend), ("attend_bwd", _Attend), ("attend_step_fwd", _AttendStep), ("group_norm_fwd", _GroupNorm),
                           ("group_norm_bwd", _GroupNorm)):
            fn = getattr(lib, f"scanscam_{name}", None)
            if fn is None:
                raise RuntimeError(f"scanscam_amd: {hip.LIB_PATH} has no scanscam_{name}: it is a build without these operators")
            fn.argtypes, fn.restype = [ctypes.POINTER(args), _p], ctypes.c_int
        for name, args, more in (("attend_saved", _Attend, []), ("attend_workspace", _Attend, [ctypes.c_int]), ("group_norm_workspace", _GroupNorm, [])):
            fn = getattr(lib, f"scanscam_{name}_bytes")
            fn.argtypes, fn.restype = [ctypes.POINTER(args)] + more, _size
        _entry_points = lib
    return _entry_points


def _bind_native():
    """The host path in native code, autograd nodes included (csrc/torch_binding.cpp), or ``None`` where it or the library is a build without
    these operators; calls then go through the functions below, several times as slowly on the host."""
    native = state_space._native
    if native is None or not hasattr(native, "bind_attention"):
        return None
    try:
        lib = _lib()
    except RuntimeError:
        return None
    native.bind_attention(*(ctypes.cast(fn, _p).value for fn in (
        lib.scanscam_attend_fwd, lib.scanscam_attend_bwd, lib.scanscam_attend_workspace_bytes, lib.scanscam_attend_step_fwd, lib.scanscam_group_norm_fwd,
        lib.scanscam_group_norm_bwd, lib.scanscam_group_norm_workspace_bytes, lib.scanscam_attend_saved_bytes)))
    return native


_native = _bind_native()


def _launching(what: str):
    """The library, for a call that launches kernels (what records ATen calls only is refused)."""
    state_space._launching(what)
    return _lib()


def _number(what: str, name: str, value) -> float:
    if isinstance(value, torch.Tensor) and value.requires_grad and torch.is_grad_enabled():
        raise TypeError(f"{what}: {name} is a number and has no gradient, got a tensor that requires one")
    return float(value)


# --------------------------------------------------------------------------------------------------------- linear attention
def _check_heads(what: str, q, k, v, decay, lead: int) -> None:
    """``lead``: 2 for [batch, T, heads, ...], 1 for [rows, heads, ...]."""
    kind = "[batch, T, heads, channels]" if lead == 2 else "[rows, heads, channels]"
    if q.dim() != lead + 2 or v.dim() != lead + 2:
        raise AssertionError(f"{what}: q, k and v must be {kind}, got shapes {tuple(q.shape)}, {tuple(k.shape)} and {tuple(v.shape)}")
    groups, K, heads, V = *q.shape[lead:], *v.shape[lead:]
    if not 1 <= K <= _MOST_HEAD or not 1 <= V <= _MOST_HEAD:
        raise AssertionError(f"{what}: a head has 1 to {_MOST_HEAD} channels, got {K} of q and k and {V} of v")
    if groups < 1 or heads % groups:
        raise AssertionError(f"{what}: {heads} heads of v are not shared out evenly to {groups} of q and k")
    _check_types(what, v, (("q", q), ("k", k)), (("decay", decay),))
    _check_shape(what, "k", k, q.shape)
    _check_shape(what, "q", q, (*v.shape[:lead], groups, K))
    if decay is not None and decay.dim() != 1:
        _check_shape(what, "decay", decay, v.shape[:lead + 1])
    else:
        _check_shape(what, "decay", decay, (heads,))


def linear_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, decay: Optional[torch.Tensor] = None, *, scale: float = 1.0,
                     state: Optional[torch.Tensor] = None, offsets: Optional[torch.Tensor] = None,
                     return_state: bool = False) -> Union[torch.Tensor, Tuple[torch.Tensor, torch.Tensor]]:
    """
    Linear attention with a decay for each head::

        S[t] = exp(decay[t]) S[t-1] + k[t] v[t]^T        (for every head, K x V values)
        y[t] = scale S[t]^T q[t]

    :param q, k: [batch, T, groups, K], shared by heads / groups neighbouring heads each; 1 to 256 channels
    :param v: [batch, T, heads, V], 1 to 256 channels
    :param decay: logs of the decays, [batch, T, heads], or [heads] for one of each head, of any of the three types; none without. They are
        meant to be 0 at most (-infinity forgets everything); above, states grow as far as float32 holds them, and what the logs of any
        64 neighbouring tokens sum up to has to be 80 at most: where float32 does not hold its exponential results are not finite.
    :param scale: a number (to train it, multiply q with it)
    :param state: [sequences, heads, K, V] in float32, the states before the first tokens (zeros if not given)
    :param offsets: the first token of each of several packed sequences, and the end
    :param return_state: hand back the states after the last tokens as well, in float32
    :return: y, [batch, T, heads, V], or ``(y, state)``. Differentiable in every tensor but ``offsets``. Products are taken in the activations'
        type and added up in float32; what float32 results come from (states, gradients of states and float32 decays) is not rounded to 16 bits.
        Values that are not finite reach the tokens after them and nothing before them; in gradients they may also reach the neighbouring 63 tokens
        of their own head and sequence, and the decays before them.
    """
    if _traced_through():
        if v.device.type == "cuda":
            return _eager(linear_attention, q, k, v, decay, scale=scale, state=state, offsets=offsets, return_state=return_state)
    elif _native is not None and _parts == 0:
        out = _native.attend(q, k, v, decay, scale, state, offsets, return_state)  # None: a call it leaves to the code below
        if out is not None:
            return out
    what = "linear_attention"
    scale = _number(what, "scale", scale)
    _check_heads(what, q, k, v, decay, 2)
    _check_devices(what, v, (("q", q), ("k", k), ("decay", decay), ("state", state), ("offsets", offsets)))
    sequences = _check_offsets(what, v, offsets)
    heads, V, K = v.shape[2], v.shape[3], q.shape[3]
    _check_shape(what, "state", state, (sequences, heads, K, V))
    if state is not None and state.dtype != torch.float32:
        raise TypeError(f"{what}: state must be float32, got {state.dtype}")
    if v.device.type != "cuda":
        return baseline.naive_linear_attention(q, k, v, decay, scale=scale, state=state, offsets=offsets, return_state=return_state)
    _check_sizes(what, max(heads * max(K, V), q.shape[2] * K), v.shape[0] * v.shape[1], sequences)
    if _needs_node(q, k, v, decay, state):
        y, new = LinearAttention.apply(q, k, v, decay, state, offsets, scale, bool(return_state))
    else:
        y, new, _, _ = _attend_forward(q, k, v, decay, state, offsets, scale, return_state, False)
    return (y, new) if return_state else y


def _logs(decay: Optional[torch.Tensor], lead: int = 2) -> _Tokens:
    return _Tokens() if decay is None else _Tokens(decay.data_ptr(), 0, 0, 0) if decay.dim() == 1 else _tokens(decay, lead)


def _attend_args(q, k, v, decay, state, offsets, scale) -> _Attend:
    a = _Attend()
    a.batch, a.T, a.heads, a.V = v.shape
    a.groups, a.K = q.shape[2:]
    a.sequences = v.shape[0] if offsets is None else offsets.shape[0] - 1
    a.offsets, a.offsets64 = _ptr(offsets), int(offsets is not None and offsets.dtype == torch.int64)
    a.dtype, a.scale, a.parts = _TYPES[v.dtype], scale, _parts
    a.q, a.k, a.v, a.decay = _tokens(q), _tokens(k), _tokens(v), _logs(decay)
    if decay is not None:
        a.decay_dtype, a.decay_fixed = _TYPES[decay.dtype], int(decay.dim() == 1)
    a.state_in = _ptr(state)
    return a


def _seen(q, k, v, decay, state, offsets):
    """The tensors as the library takes them."""
    return _near(q), _near(k), _near(v), _unit(decay), _dense(state), _dense(offsets)


def _attend_forward(q, k, v, decay, state, offsets, scale, return_state, save):
    """``(y, new state or None, saved or None, the tensors as the library saw them)``."""
    L = _launching("linear_attention")
    with hip._on(v.device):
        seen = _seen(q, k, v, decay, state, offsets)
        a = _attend_args(*seen, scale)
        y = torch.empty(v.shape, dtype=v.dtype, device=v.device)
        a.y = _tokens(y)
        new = saved = workspace = None
        if return_state:
            new = torch.empty((a.sequences, a.heads, a.K, a.V), dtype=torch.float32, device=v.device)
            a.state_out = new.data_ptr()
        if save:
            saved = _bytes(L.scanscam_attend_saved_bytes(a), v.device)
            a.saved = _ptr(saved)
        n = L.scanscam_attend_workspace_bytes(a, hip.FORWARD)
        if n:
            workspace = _bytes(n, v.device)
            a.workspace, a.workspace_bytes = workspace.data_ptr(), n
        _raise(L.scanscam_attend_fwd(a, _stream(v.device)), "attend_fwd")
    return y, new, saved, seen


class LinearAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, decay, state, offsets, scale, return_state):
        y, new, saved, seen = _attend_forward(q, k, v, decay, state, offsets, scale, return_state, True)
        ctx.save_for_backward(*seen, saved)
        ctx.meta = _meta(*seen, saved)
        ctx.scale = scale
        ctx.set_materialize_grads(False)
        return y, new

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, gy, gnew):
        if gy is None and gnew is None:
            return (None,) * 8
        kept = ctx.saved_tensors
        _check_saved("linear_attention", gy if gy is not None else gnew, dict(zip(("q", "k", "v", "decay", "state", "offsets", "saved states"), kept)), ctx.meta)
        q, k, v, decay, state, offsets = seen = _seen(*kept[:6])  # (a hook on saved tensors may lay out what it gives back in its own way)
        L = _launching("linear_attention")
        with hip._on(v.device):
            gy = _near(gy) if gy is not None else torch.zeros(v.shape, dtype=v.dtype, device=v.device)
            gnew = _dense(gnew)
            a = _attend_args(*seen, ctx.scale)
            gq, gk, gv = (torch.empty(t.shape, dtype=t.dtype, device=v.device) for t in (q, k, v))
            gdecay = torch.empty(decay.shape, dtype=torch.float32, device=v.device) if ctx.needs_input_grad[3] else None
            gstate = torch.empty(state.shape, dtype=torch.float32, device=v.device) if ctx.needs_input_grad[4] else None
            a.gy, a.gq, a.gk, a.gv = (_tokens(t) for t in (gy, gq, gk, gv))
            saved = _dense(kept[6])
            a.gdecay, a.gstate_out, a.gstate_in, a.saved = _ptr(gdecay), _ptr(gnew), _ptr(gstate), _ptr(saved)
            n = L.scanscam_attend_workspace_bytes(a, hip.BACKWARD)
            workspace = _bytes(n, v.device)
            a.workspace, a.workspace_bytes = _ptr(workspace), n
            _raise(L.scanscam_attend_bwd(a, _stream(v.device)), "attend_bwd")
            return gq, gk, gv, None if gdecay is None else gdecay.to(decay.dtype), gstate, None, None, None


def linear_attention_step(state: torch.Tensor, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, decay: Optional[torch.Tensor] = None, *,
                          scale: float = 1.0, slots: Optional[torch.Tensor] = None) -> torch.Tensor:
    """
    One token of each of several sequences: ``linear_attention``'s formulas, from and into their states.

    :param state: [slots, heads, K, V] in float32, contiguous, updated in place
    :param q, k: [rows, groups, K]; v: [rows, heads, V]; decay: [rows, heads] or [heads]; slots as for ``selective_scan_step``
    :return: y, [rows, heads, V]. Not differentiable.
    """
    if _traced_through():
        if v.device.type == "cuda":
            return _eager(linear_attention_step, state, q, k, v, decay, scale=scale, slots=slots)
    elif _native is not None:
        out = _native.attend_step(state, q, k, v, decay, scale, slots)
        if out is not None:
            return out
    what = "linear_attention_step"
    scale = _number(what, "scale", scale)
    _check_heads(what, q, k, v, decay, 1)
    _check_devices(what, v, (("state", state), ("q", q), ("k", k), ("decay", decay), ("slots", slots)))
    rows, heads, V = v.shape
    if state.dim() != 4:
        raise AssertionError(f"{what}: state must be [slots, heads, K, V], got shape {tuple(state.shape)}")
    _check_shape(what, "state", state, (state.shape[0], heads, q.shape[2], V))
    if state.dtype != torch.float32:
        raise TypeError(f"{what}: state must be float32, got {state.dtype}")
    _check_slots(what, rows, state, slots)
    _check_in_place(what, state)
    if _wants_grad(q, k, v, decay) or _has_tangent(state, q, k, v, decay):
        raise RuntimeError(f"{what}: a single token's step has no gradient; call it under torch.no_grad()")
    if v.device.type != "cuda":
        return baseline.naive_linear_attention_step(state, q, k, v, decay, scale=scale, slots=slots)
    _check_sizes(what, heads * max(q.shape[2], V), rows)
    if torch.jit.is_tracing():
        return LinearAttentionStep.apply(state, q, k, v, decay, slots, scale)
    return _attend_step(state, q, k, v, decay, slots, scale)


def _attend_step(state, q, k, v, decay, slots, scale):
    L = _launching("linear_attention_step")
    with hip._on(v.device):
        q, k, v, decay, slots = _unit(q), _unit(k), _unit(v), _unit(decay), _dense(slots)
        (rows, heads, V), (groups, K) = v.shape, q.shape[1:]
        y = torch.empty(v.shape, dtype=v.dtype, device=v.device)
        a = _AttendStep(rows, heads, groups, K, V, state.shape[0], _ptr(slots), int(slots is not None and slots.dtype == torch.int64), _TYPES[v.dtype],
                        0 if decay is None else _TYPES[decay.dtype], scale, *(_tokens_of_rows(t) for t in (q, k, v, y)), _logs(decay, 1), state.data_ptr())
        _raise(L.scanscam_attend_step_fwd(a, _stream(v.device)), "attend_step_fwd")
    torch.autograd.graph.increment_version(state)  # (written in place)
    return y


def _tokens_of_rows(t: torch.Tensor) -> _Tokens:
    return _Tokens(t.data_ptr(), 0, t.stride(0), t.stride(1))


class LinearAttentionStep(torch.autograd.Function):
    """What a trace records of a step; there is no gradient."""

    @staticmethod
    def forward(ctx, state, q, k, v, decay, slots, scale):
        y = _attend_step(state, q, k, v, decay, slots, scale)
        ctx.mark_non_differentiable(y)
        return y


# ----------------------------------------------------------------------------------------------------------------- group norm
def group_norm(x: torch.Tensor, groups: int, weight: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None,
               z: Optional[torch.Tensor] = None, *, eps: float = 1e-5, activation: Optional[str] = None) -> torch.Tensor:
    """
    Norm of every group of a token's channels (the heads of an attention's output), with an activation and a gate::

        u = (x - mean) / sqrt(variance + eps) * weight + bias        (mean and variance of the group's channels)
        y = act(u) * silu(z)

    :param x: [..., channels], channels shared out to the groups in order, up to 8192 each
    :param weight, bias: [channels], optional; z: gates of x's shape and type, optional
    :param activation: None or "silu"
    :return: y, of x's shape and type. Differentiable in every tensor. Squares are added up in float32: rows of values past some 1e19 come out
        as the bias alone.
    """
    if _traced_through():
        if x.device.type == "cuda":
            return _eager(group_norm, x, groups, weight, bias, z, eps=eps, activation=activation)
    elif _native is not None:
        out = _native.group_norm(x, groups, weight, bias, z, eps, activation)
        if out is not None:
            return out
    what = "group_norm"
    groups, eps = operator.index(groups), _number(what, "eps", eps)
    if x.dim() < 1 or groups < 1 or x.shape[-1] % groups:
        raise AssertionError(f"{what}: x must be [..., channels] with channels shared out evenly to the groups, got shape {tuple(x.shape)} and {groups} groups")
    if x.shape[-1] // groups > _MOST_GROUP:
        raise AssertionError(f"{what}: a group has up to {_MOST_GROUP} channels, got {x.shape[-1] // groups}")
    _check_activation(what, activation)
    _check_types(what, x, (("z", z),), (("weight", weight), ("bias", bias)))
    _check_devices(what, x, (("weight", weight), ("bias", bias), ("z", z)))
    for name, t, shape in (("weight", weight, x.shape[-1:]), ("bias", bias, x.shape[-1:]), ("z", z, x.shape)):
        _check_shape(what, name, t, shape)
    if x.device.type != "cuda":
        return baseline.naive_group_norm(x, groups, weight, bias, z, eps=eps, activation=activation)
    _check_sizes(what, x.shape[-1], x.shape[:-1].numel())
    if _needs_node(x, weight, bias, z):
        return GroupNorm.apply(x, groups, weight, bias, z, eps, activation)
    return _group_norm_forward(x, groups, weight, bias, z, eps, activation)[0]


def _group_norm_args(x, groups, weight, bias, z, eps, activation) -> _GroupNorm:
    """``x``, ``z``: rows."""
    a = _GroupNorm()
    a.rows, a.channels = x.shape
    a.groups, a.eps, a.dtype, a.activation = groups, eps, _TYPES[x.dtype], _ACTIVATIONS[activation]
    a.x, a.x_stride, a.weight, a.bias = x.data_ptr(), x.stride(0), _param(weight), _param(bias)
    if z is not None:
        a.z, a.z_stride = z.data_ptr(), z.stride(0)
    return a


def _group_norm_forward(x, groups, weight, bias, z, eps, activation):
    """``(y, the tensors as the library saw them)``."""
    L = _launching("group_norm")
    with hip._on(x.device):
        seen = _rows(x), _dense(weight), _dense(bias), _rows(z)
        a = _group_norm_args(seen[0], groups, *seen[1:], eps, activation)
        y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
        a.y = y.data_ptr()
        _raise(L.scanscam_group_norm_fwd(a, _stream(x.device)), "group_norm_fwd")
    return y, seen


class GroupNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, groups, weight, bias, z, eps, activation):
        y, seen = _group_norm_forward(x, groups, weight, bias, z, eps, activation)
        ctx.save_for_backward(*seen)
        ctx.meta = _meta(*seen)
        ctx.call = groups, eps, activation
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, gy):
        kept = ctx.saved_tensors
        _check_saved("group_norm", gy, dict(zip(("x", "weight", "bias", "z"), kept)), ctx.meta)
        groups, eps, activation = ctx.call
        L = _launching("group_norm")
        with hip._on(gy.device):
            x, weight, bias, z = _rows(kept[0]), _dense(kept[1]), _dense(kept[2]), _rows(kept[3])
            gy = gy.contiguous()
            a = _group_norm_args(x, groups, weight, bias, z, eps, activation)
            gx, gz = (None if t is None else torch.empty(gy.shape, dtype=gy.dtype, device=gy.device) for t in (x, z))
            gweight, gbias = (None if t is None else torch.empty(t.shape, dtype=torch.float32, device=gy.device) for t in (weight, bias))
            a.gy, a.gx, a.gz, a.gweight, a.gbias = gy.data_ptr(), gx.data_ptr(), _ptr(gz), _ptr(gweight), _ptr(gbias)
            n = L.scanscam_group_norm_workspace_bytes(a)
            workspace = _bytes(n, gy.device)
            a.workspace, a.workspace_bytes = _ptr(workspace), n
            _raise(L.scanscam_group_norm_bwd(a, _stream(gy.device)), "group_norm_bwd")
            cast = lambda g, t: g if g is None else g.to(t.dtype)  # noqa: E731
            return gx, None, cast(gweight, weight), cast(gbias, bias), gz, None, None
