"""
The operators of a state space layer in a language model: the selective scan, the short causal convolution before it
and the root-mean-square norm with the residual's addition, over whole sequences with gradients and for single tokens.

Activations are tokens-first, ``[batch, T, channels]``, as linear layers produce and consume them, in float32,
bfloat16 or float16 (arithmetic in float32); views with a unit stride along the channels -- parts of a projection -- are
taken as they are, others are copied first. Parameters may be of any of the three types. Packed sequences are one batch
element whose tokens belong to sequence ``s`` from ``offsets[s]`` up to ``offsets[s + 1]`` (an int32 or int64 tensor of one entry
more than there are sequences, on the same device, from 0 to T, not decreasing; it is not looked at on the host).

GPU tensors run the kernels of ``libscanscam_hip.so`` (C ABI in ``include/scanscam_ops.h``) on the current stream and nothing
else, up to 2^20 channels and 2^31 - 2^20 tokens, rows or sequences a call; CPU tensors take the loops of ``scanscam_amd.baseline``. Calls can be recorded by
``torch.jit.trace`` and by graphs, and made from functions under ``torch.compile``, whose graph they break; ``make_fx`` and forward-mode derivatives
are refused on the GPU. None of this has a counterpart in the reference, whose one
operator is the scan.
"""
import ctypes
import sys
from typing import Optional, Tuple, Union

import torch
from torch.autograd import forward_ad

from . import baseline, hip

_TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
_EIGHT = {torch.int8: 16, torch.float8_e4m3fn: 17}
_ACTIVATIONS = {None: 0, "silu": 1}
_MOST_STATES, _MOST_TAPS, _MOST_NORM_CHANNELS, _MOST_TOKEN_STRIDE = 256, 8, 32768, 1 << 22
_MOST_CHANNELS, _MOST_TOKENS = 1 << 20, (1 << 31) - (1 << 20)

_p, _i32, _i64, _f32, _size = ctypes.c_void_p, ctypes.c_int32, ctypes.c_int64, ctypes.c_float, ctypes.c_size_t


class _Tokens(ctypes.Structure):
    _fields_ = [("p", _p), ("batch", _i64), ("token", _i64), ("group", _i64)]


class _Param(ctypes.Structure):
    _fields_ = [("p", _p), ("dtype", _i32), ("unused", _i32)]


class _Selective(ctypes.Structure):
    _fields_ = ([(n, _i64) for n in ("batch", "T", "sequences", "channels", "groups", "N")] + [("offsets", _p)] +
                [(n, _i32) for n in ("offsets64", "dtype", "softplus", "parts")] +
                [(n, _Tokens) for n in ("x", "dt", "B", "C", "z", "y")] + [(n, _Param) for n in ("A", "D", "dt_bias")] +
                [(n, _p) for n in ("state_in", "state_out", "saved")] +
                [(n, _Tokens) for n in ("gy", "gx", "gdt", "gB", "gC", "gz")] +
                [(n, _p) for n in ("gA", "gD", "gdt_bias", "gstate_out", "gstate_in", "workspace")] + [("workspace_bytes", _size)])


class _SelectiveStep(ctypes.Structure):
    _fields_ = ([(n, _i64) for n in ("rows", "channels", "groups", "N", "slots")] + [("slot", _p)] +
                [(n, _i32) for n in ("slot64", "dtype", "softplus", "unused")] +
                [(n, _Tokens) for n in ("x", "dt", "B", "C", "z", "y")] + [(n, _Param) for n in ("A", "D", "dt_bias")] + [("state", _p)])


class _Conv(ctypes.Structure):
    _fields_ = ([(n, _i64) for n in ("batch", "T", "sequences", "channels", "K")] + [("offsets", _p)] +
                [(n, _i32) for n in ("offsets64", "dtype", "activation", "unused")] + [("x", _Tokens), ("y", _Tokens)] +
                [("weight", _Param), ("bias", _Param), ("state_in", _p), ("state_out", _p), ("gy", _Tokens), ("gx", _Tokens)] +
                [(n, _p) for n in ("gweight", "gbias", "gstate_out", "gstate_in", "workspace")] + [("workspace_bytes", _size)])


class _ConvStep(ctypes.Structure):
    _fields_ = ([(n, _i64) for n in ("rows", "channels", "K", "slots")] + [("slot", _p)] +
                [(n, _i32) for n in ("slot64", "dtype", "activation", "unused")] + [("x", _Tokens), ("y", _Tokens)] +
                [("weight", _Param), ("bias", _Param), ("state", _p)])


class _Norm(ctypes.Structure):
    _fields_ = ([(n, _i64) for n in ("rows", "channels", "x_stride", "residual_stride")] + [("x", _p), ("residual", _p), ("weight", _Param)] +
                [(n, _p) for n in ("y", "sum", "rstd", "scale")] + [("eps", _f32)] +
                [(n, _i32) for n in ("dtype", "residual_dtype", "out_dtype")] +
                [(n, _p) for n in ("gy", "gsum", "gx", "gresidual", "gweight", "workspace")] + [("workspace_bytes", _size)])


_entry_points = None
# Parts of time that the selective scan's workgroups share a sequence out in; 0: the library chooses (the tests force others).
_parts = 0


def _lib():
    """The library with these operators' entry points bound; raises where they are missing."""
    global _entry_points
    if _entry_points is None:
        lib = hip.lib()
        for name, args in (("selective_fwd", _Selective), ("selective_bwd", _Selective), ("selective_step_fwd", _SelectiveStep),
                           ("conv_fwd", _Conv), ("conv_bwd", _Conv), ("conv_step_fwd", _ConvStep),
                           ("norm_fwd", _Norm), ("norm_bwd", _Norm)):
            fn = getattr(lib, f"scanscam_{name}", None)
            if fn is None:
                raise RuntimeError(f"scanscam_amd: {hip.LIB_PATH} has no scanscam_{name}: it is a build without these operators")
            fn.argtypes, fn.restype = [ctypes.POINTER(args), _p], ctypes.c_int
        for name, args, more in (("selective_saved", _Selective, []), ("selective_workspace", _Selective, [ctypes.c_int]),
                                 ("conv_workspace", _Conv, []), ("norm_workspace", _Norm, [])):
            fn = getattr(lib, f"scanscam_{name}_bytes")
            fn.argtypes, fn.restype = [ctypes.POINTER(args)] + more, _size
        _entry_points = lib
    return _entry_points


def _launching(what: str):
    """The library, for a call that launches kernels. make_fx records ATen calls, of which a launch is none: it would record outputs that
    nothing writes."""
    recorder = sys.modules.get("torch.fx.experimental.proxy_tensor")  # (where nothing has imported it nothing records)
    if recorder is not None and recorder.get_proxy_mode() is not None:
        raise RuntimeError(f"{what}: make_fx cannot record this call, whose kernels are no ATen operators")
    return _lib()


def _bind_native():
    """The host path in native code, autograd nodes included (csrc/torch_binding.cpp), or ``None`` where it is not built or the library is
    a build without these operators; calls then go through the functions below, three times as slowly on the host."""
    if hip._native is None or not hasattr(hip._native, "bind_operators"):
        return None
    try:
        lib = _lib()
    except RuntimeError:
        return None
    hip._native.bind_operators(*(ctypes.cast(fn, _p).value for fn in (
        lib.scanscam_selective_fwd, lib.scanscam_selective_workspace_bytes, lib.scanscam_selective_step_fwd, lib.scanscam_conv_fwd,
        lib.scanscam_conv_step_fwd, lib.scanscam_norm_fwd, lib.scanscam_selective_bwd, lib.scanscam_selective_saved_bytes,
        lib.scanscam_conv_bwd, lib.scanscam_conv_workspace_bytes, lib.scanscam_norm_bwd, lib.scanscam_norm_workspace_bytes)))
    return hip._native


_native = _bind_native()


def _raise(rc: int, what: str) -> None:
    if rc != 0:
        raise RuntimeError(f"scanscam_{what}: {hip.strerror(rc)}")


def _stream(device: torch.device) -> int:
    return torch.cuda.current_stream(device).cuda_stream


# ---------------------------------------------------------------------------------------------------------------- compiled callers
_outside = {}


def _eager(fn, *args, **kwargs):
    """A call from a function that torch.compile traces: it breaks the graph there and runs as it does everywhere else. (Traced through, it
    would come to the library's entry points, which no graph can hold.)"""
    if fn not in _outside:
        _outside[fn] = torch.compiler.disable(fn)
    return _outside[fn](*args, **kwargs)


_eager._torchdynamo_disable = True  # (what torch.compiler.disable marks, without its import of the compiler)


_traced_through = torch.compiler.is_dynamo_compiling


# --------------------------------------------------------------------------------------------------------- checks of arguments
def _check_types(what: str, first: torch.Tensor, tensors, params) -> None:
    if first.dtype not in _TYPES:
        raise TypeError(f"{what}: unsupported dtype {first.dtype}; supported: float32, bfloat16, float16")
    for name, t in tensors:
        if t is not None and t.dtype != first.dtype:
            raise TypeError(f"{what}: {name} is {t.dtype}, the activations are {first.dtype}")
    for name, t in params:
        if t is not None and t.dtype not in _TYPES:
            raise TypeError(f"{what}: unsupported dtype {t.dtype} of {name}; supported: float32, bfloat16, float16")


def _check_devices(what: str, first: torch.Tensor, tensors) -> None:
    for name, t in tensors:
        if t is not None and t.device != first.device:
            raise RuntimeError(f"{what}: {name} is on {t.device}, the activations on {first.device}")


def _check_shape(what: str, name: str, t: Optional[torch.Tensor], shape) -> None:
    if t is not None and tuple(t.shape) != tuple(shape):
        raise AssertionError(f"{what}: {name} must have shape {tuple(shape)}, got {tuple(t.shape)}")


def _check_sizes(what: str, channels: int, tokens: int, sequences: int = 0) -> None:
    """What one call on the GPU takes (CPU tensors have no such limits)."""
    if channels > _MOST_CHANNELS or max(tokens, sequences) >= _MOST_TOKENS:
        raise AssertionError(f"{what}: a call takes up to {_MOST_CHANNELS} channels and fewer than {_MOST_TOKENS} tokens, rows or sequences, "
                             f"got {channels} channels, {tokens} tokens" + (f", {sequences} sequences" if sequences else ""))


def _check_offsets(what: str, x: torch.Tensor, offsets: Optional[torch.Tensor]) -> int:
    """The number of sequences."""
    if offsets is None:
        return x.shape[0]
    if offsets.dtype not in (torch.int32, torch.int64):
        raise TypeError(f"{what}: offsets must be int32 or int64, got {offsets.dtype}")
    if offsets.dim() != 1 or offsets.shape[0] < 2 or x.shape[0] != 1:
        raise AssertionError(f"{what}: offsets are [sequences + 1] with one batch element, got {tuple(offsets.shape)} and batch {x.shape[0]}")
    return offsets.shape[0] - 1


def _check_slots(what: str, rows: int, state: torch.Tensor, slots: Optional[torch.Tensor]) -> None:
    if slots is None:
        if state.shape[0] != rows:
            raise AssertionError(f"{what}: without slots, state must have a row for each of the {rows} tokens, got {state.shape[0]}")
        return
    if slots.dtype not in (torch.int32, torch.int64):
        raise TypeError(f"{what}: slots must be int32 or int64, got {slots.dtype}")
    _check_shape(what, "slots", slots, (rows,))


def _check_in_place(what: str, state: torch.Tensor) -> None:
    if not state.is_contiguous():
        raise RuntimeError(f"{what}: state is updated in place and must be contiguous")
    if state.requires_grad and torch.is_grad_enabled():
        raise RuntimeError(f"{what}: a single token's step has no gradient; the state requires one")


def _check_activation(what: str, activation: Optional[str]) -> None:
    if activation not in _ACTIVATIONS:
        raise ValueError(f"{what}: activation must be None or 'silu', got {activation!r}")


def _grouped(t: torch.Tensor) -> torch.Tensor:
    """B or C of one group, ``[..., N]``, as ``[..., 1, N]``."""
    return t.unsqueeze(-2)


# What was saved for a backward pass, and what a hook on saved tensors gives back for it: in a layout of its own, but the kernels take addresses.
def _meta(*tensors):
    return [None if t is None else (t.shape, t.dtype) for t in tensors]


def _check_saved(what: str, grad: torch.Tensor, tensors: dict, meta) -> None:
    for (name, t), kept in zip(tensors.items(), meta):
        if t is not None and (t.device != grad.device or (t.shape, t.dtype) != kept):
            raise RuntimeError(f"{what}: {name} was saved for the backward pass as {kept[1]} {tuple(kept[0])} on {grad.device} and came back as "
                               f"{t.dtype} {tuple(t.shape)} on {t.device}")


# ---------------------------------------------------------------------------------------------------------- views for the library
def _unit(t: Optional[torch.Tensor]) -> Optional[torch.Tensor]:
    """The tensor itself where its last dimension is unit-stride, else a copy."""
    if t is None or t.shape[-1] == 1 or t.stride(-1) == 1:
        return t
    return t.contiguous()


def _near(t: Optional[torch.Tensor]) -> Optional[torch.Tensor]:
    """The same for the selective scan of whole sequences, whose kernels take tokens at most so far apart; B and C of very many groups
    come group by group then."""
    t = _unit(t)
    if t is None or t.shape[1] <= 1 or t.stride(1) < _MOST_TOKEN_STRIDE:
        return t
    t = t.contiguous()
    return t if t.stride(1) < _MOST_TOKEN_STRIDE else t.permute(2, 0, 1, 3).contiguous().permute(1, 2, 0, 3)


def _empty_near(t: Optional[torch.Tensor]) -> Optional[torch.Tensor]:
    """An output of t's shape that the selective scan takes."""
    if t is None:
        return None
    if t.dim() < 4 or t.shape[2] * t.shape[3] < _MOST_TOKEN_STRIDE:
        return torch.empty(t.shape, dtype=t.dtype, device=t.device)
    batch, T, groups, N = t.shape
    return torch.empty((groups, batch, T, N), dtype=t.dtype, device=t.device).permute(1, 2, 0, 3)


def _tokens(t: Optional[torch.Tensor], lead: int = 2) -> _Tokens:
    """``lead``: 2 for [batch, T, ...], 1 for [rows, ...]."""
    if t is None:
        return _Tokens()
    st = t.stride()
    batch, token = (st[0], st[1]) if lead == 2 else (0, st[0])
    if t.shape[lead - 1] == 1:
        token = 0  # (a single token's distance to the next may be anything)
    return _Tokens(t.data_ptr(), batch, token, st[lead] if t.dim() > lead + 1 else 0)


def _param(t: Optional[torch.Tensor]) -> _Param:
    return _Param() if t is None else _Param(t.data_ptr(), _TYPES[t.dtype], 0)


def _ptr(t: Optional[torch.Tensor]) -> Optional[int]:
    return None if t is None else t.data_ptr()


def _dense(t: Optional[torch.Tensor]) -> Optional[torch.Tensor]:
    return None if t is None else t.contiguous()


def _bytes(n: int, device: torch.device) -> Optional[torch.Tensor]:
    return torch.empty(n, dtype=torch.uint8, device=device) if n else None


def _wants_grad(*tensors) -> bool:
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)


def _has_tangent(*tensors) -> bool:
    """Whether a forward-mode derivative is asked for, which no kernel here has: calls with gradients go through their autograd
    function, which refuses it as scan()'s does, and the others refuse it themselves. (The CPU's loops have them.)"""
    if getattr(forward_ad, "_current_level", 0) < 0:  # (no call under dual_level() is under way: unpack_dual() would look there first)
        return False
    return any(t is not None and t.device.type == "cuda" and forward_ad.unpack_dual(t).tangent is not None for t in tensors)


def _needs_node(*tensors) -> bool:
    """Whether a call has to go through its autograd function: for gradients, and where torch.jit.trace records it, which sees the function but
    not a launch (it would record the allocation of the outputs and nothing that writes them)."""
    return _wants_grad(*tensors) or _has_tangent(*tensors) or torch.jit.is_tracing()


# -------------------------------------------------------------------------------------------------------------------- selective scan
def selective_scan(x: torch.Tensor, dt: torch.Tensor, A: torch.Tensor, B: torch.Tensor, C: torch.Tensor,
                   D: Optional[torch.Tensor] = None, z: Optional[torch.Tensor] = None, dt_bias: Optional[torch.Tensor] = None, *,
                   softplus: bool = False, state: Optional[torch.Tensor] = None, offsets: Optional[torch.Tensor] = None,
                   return_state: bool = False) -> Union[torch.Tensor, Tuple[torch.Tensor, torch.Tensor]]:
    """
    The selective scan of a state space layer. With ``d = dt + dt_bias``, softplus of it where ``softplus`` is set::

        h[t] = exp(d[t] A) h[t-1] + d[t] x[t] B[t]        (for every channel, N states)
        y[t] = (sum over the states of C[t] h[t] + D x[t]) * silu(z[t])

    :param x, dt, z: [batch, T, channels] inputs, step sizes and (optional) gates
    :param A: [channels, N], 1 to 256 states a channel
    :param B, C: [batch, T, N], or [batch, T, groups, N] shared by channels / groups neighbouring channels each
    :param D, dt_bias: [channels], optional
    :param state: [sequences, channels, N] in float32, the states before the first tokens (zeros if not given)
    :param offsets: the first token of each of several packed sequences, and the end
    :param return_state: hand back the states after the last tokens as well, in float32
    :return: y, or ``(y, state)``. Differentiable in every tensor but ``offsets``.
    """
    if _traced_through():
        if x.device.type == "cuda":
            return _eager(selective_scan, x, dt, A, B, C, D, z, dt_bias, softplus=softplus, state=state, offsets=offsets, return_state=return_state)
    elif _native is not None and _parts == 0:
        out = _native.selective(x, dt, A, B, C, D, z, dt_bias, softplus, state, offsets, return_state)  # None: a call it leaves to the code below
        if out is not None:
            return out
    what = "selective_scan"
    if x.dim() != 3:
        raise AssertionError(f"{what}: x must be [batch, T, channels], got shape {tuple(x.shape)}")
    batch, T, channels = x.shape
    if A.dim() != 2 or B.dim() not in (3, 4) or not 1 <= A.shape[1] <= _MOST_STATES:
        raise AssertionError(f"{what}: A must be [channels, 1 to {_MOST_STATES} states] and B [batch, T, (groups,) states], got {tuple(A.shape)} and {tuple(B.shape)}")
    N, groups = A.shape[1], B.shape[2] if B.dim() == 4 else 1
    if groups < 1 or channels % groups:
        raise AssertionError(f"{what}: {channels} channels are not shared out evenly to {groups} groups")
    _check_types(what, x, (("dt", dt), ("B", B), ("C", C), ("z", z)), (("A", A), ("D", D), ("dt_bias", dt_bias)))
    _check_devices(what, x, (("dt", dt), ("A", A), ("B", B), ("C", C), ("D", D), ("z", z), ("dt_bias", dt_bias), ("state", state), ("offsets", offsets)))
    sequences = _check_offsets(what, x, offsets)
    for name, t, shape in (("dt", dt, x.shape), ("z", z, x.shape), ("A", A, (channels, N)), ("C", C, B.shape), ("D", D, (channels,)),
                           ("dt_bias", dt_bias, (channels,)), ("state", state, (sequences, channels, N)),
                           ("B", B, (batch, T, groups, N) if B.dim() == 4 else (batch, T, N))):
        _check_shape(what, name, t, shape)
    if state is not None and state.dtype != torch.float32:
        raise TypeError(f"{what}: state must be float32, got {state.dtype}")
    if x.device.type != "cuda":
        return baseline.naive_selective_scan(x, dt, A, B, C, D, z, dt_bias, softplus=softplus, state=state, offsets=offsets, return_state=return_state)
    _check_sizes(what, channels, batch * T, sequences)
    if B.dim() == 3:
        B, C = _grouped(B), _grouped(C)
    if _needs_node(x, dt, A, B, C, D, z, dt_bias, state):
        y, new = SelectiveScan.apply(x, dt, A, B, C, D, z, dt_bias, state, offsets, bool(softplus), bool(return_state))
    else:
        y, new, _, _ = _selective_forward(x, dt, A, B, C, D, z, dt_bias, state, offsets, softplus, return_state, False)
    return (y, new) if return_state else y


def _selective_args(x, dt, A, B, C, D, z, dt_bias, state, offsets, softplus) -> _Selective:
    a = _Selective()
    a.batch, a.T, a.channels = x.shape
    a.sequences = x.shape[0] if offsets is None else offsets.shape[0] - 1
    a.groups, a.N = B.shape[2], A.shape[1]
    a.offsets, a.offsets64 = _ptr(offsets), int(offsets is not None and offsets.dtype == torch.int64)
    a.dtype, a.softplus, a.parts = _TYPES[x.dtype], int(softplus), _parts
    a.x, a.dt, a.B, a.C, a.z = (_tokens(t) for t in (x, dt, B, C, z))
    a.A, a.D, a.dt_bias = _param(A), _param(D), _param(dt_bias)
    a.state_in = _ptr(state)
    return a


def _selective_forward(x, dt, A, B, C, D, z, dt_bias, state, offsets, softplus, return_state, save):
    """``(y, new state or None, saved or None, the tensors as the library saw them)``."""
    L = _launching("selective_scan")
    with hip._on(x.device):
        seen = (_near(x), _near(dt), _dense(A), _near(B), _near(C), _dense(D), _near(z), _dense(dt_bias), _dense(state), _dense(offsets))
        a = _selective_args(*seen, softplus)
        y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
        a.y = _tokens(y)
        new = saved = workspace = None
        if return_state:
            new = torch.empty((a.sequences, a.channels, a.N), dtype=torch.float32, device=x.device)
            a.state_out = new.data_ptr()
        if save:
            saved = _bytes(L.scanscam_selective_saved_bytes(a), x.device)
            a.saved = _ptr(saved)
        n = L.scanscam_selective_workspace_bytes(a, hip.FORWARD)
        if n:
            workspace = _bytes(n, x.device)
            a.workspace, a.workspace_bytes = workspace.data_ptr(), n
        _raise(L.scanscam_selective_fwd(a, _stream(x.device)), "selective_fwd")
    return y, new, saved, seen


class SelectiveScan(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, dt, A, B, C, D, z, dt_bias, state, offsets, softplus, return_state):
        y, new, saved, seen = _selective_forward(x, dt, A, B, C, D, z, dt_bias, state, offsets, softplus, return_state, True)
        ctx.save_for_backward(*seen, saved)
        ctx.meta = _meta(*seen, saved)
        ctx.softplus = softplus
        ctx.set_materialize_grads(False)
        return y, new

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, gy, gnew):
        if gy is None and gnew is None:
            return (None,) * 12
        x, dt, A, B, C, D, z, dt_bias, state, offsets, saved = ctx.saved_tensors
        given = {"x": x, "dt": dt, "A": A, "B": B, "C": C, "D": D, "z": z, "dt_bias": dt_bias, "state": state, "offsets": offsets, "saved states": saved}
        _check_saved("selective_scan", gy if gy is not None else gnew, given, ctx.meta)
        # (a hook on saved tensors may lay out what it gives back in its own way)
        x, dt, B, C, z = (_near(t) for t in (x, dt, B, C, z))
        A, D, dt_bias, state, offsets, saved = (_dense(t) for t in (A, D, dt_bias, state, offsets, saved))
        seen = x, dt, A, B, C, D, z, dt_bias, state, offsets
        L = _launching("selective_scan")
        with hip._on(x.device):
            gy = _near(gy) if gy is not None else torch.zeros(x.shape, dtype=x.dtype, device=x.device)
            gnew = _dense(gnew)
            a = _selective_args(*seen, ctx.softplus)
            new = lambda t, dtype=None: None if t is None else torch.empty(t.shape, dtype=dtype or t.dtype, device=x.device)  # noqa: E731
            gx, gdt, gB, gC, gz = (_empty_near(t) for t in (x, dt, B, C, z))
            gA, gD, gbias = (new(t, torch.float32) for t in (A, D, dt_bias))
            gstate = new(state) if ctx.needs_input_grad[8] else None
            a.gy, a.gx, a.gdt, a.gB, a.gC, a.gz = (_tokens(t) for t in (gy, gx, gdt, gB, gC, gz))
            a.gA, a.gD, a.gdt_bias, a.gstate_out, a.gstate_in, a.saved = (_ptr(t) for t in (gA, gD, gbias, gnew, gstate, saved))
            n = L.scanscam_selective_workspace_bytes(a, hip.BACKWARD)
            workspace = _bytes(n, x.device)
            a.workspace, a.workspace_bytes = _ptr(workspace), n
            _raise(L.scanscam_selective_bwd(a, _stream(x.device)), "selective_bwd")
            cast = lambda g, t: g if g is None or t.dtype == torch.float32 else g.to(t.dtype)  # noqa: E731
            return gx, gdt, cast(gA, A), gB, gC, cast(gD, D), gz, cast(gbias, dt_bias), gstate, None, None, None


def selective_scan_step(state: torch.Tensor, x: torch.Tensor, dt: torch.Tensor, A: torch.Tensor, B: torch.Tensor, C: torch.Tensor,
                        D: Optional[torch.Tensor] = None, z: Optional[torch.Tensor] = None, dt_bias: Optional[torch.Tensor] = None, *,
                        softplus: bool = False, slots: Optional[torch.Tensor] = None) -> torch.Tensor:
    """
    One token of each of several sequences: ``selective_scan``'s formulas, from and into their states.

    :param state: [slots, channels, N] in float32, contiguous, updated in place
    :param x, dt, z: [rows, channels]; B, C: [rows, N] or [rows, groups, N]; the rest as for ``selective_scan``
    :param slots: [rows], the row of ``state`` of each token (row i for token i if not given; no two may be the same). A token whose
        slot is not in ``state``, such as -1, is left out: its output is zero and no state changes.
    :return: y, [rows, channels]. Not differentiable.
    """
    if _traced_through():
        if x.device.type == "cuda":
            return _eager(selective_scan_step, state, x, dt, A, B, C, D, z, dt_bias, softplus=softplus, slots=slots)
    elif _native is not None:
        out = _native.selective_step(state, x, dt, A, B, C, D, z, dt_bias, softplus, slots)
        if out is not None:
            return out
    what = "selective_scan_step"
    if x.dim() != 2 or state.dim() != 3 or A.dim() != 2 or B.dim() not in (2, 3) or not 1 <= A.shape[1] <= _MOST_STATES:
        raise AssertionError(f"{what}: x must be [rows, channels], state [slots, channels, N], A [channels, N], B [rows, (groups,) N], "
                             f"got {tuple(x.shape)}, {tuple(state.shape)}, {tuple(A.shape)} and {tuple(B.shape)}")
    (rows, channels), N, groups = x.shape, A.shape[1], B.shape[1] if B.dim() == 3 else 1
    if groups < 1 or channels % groups:
        raise AssertionError(f"{what}: {channels} channels are not shared out evenly to {groups} groups")
    _check_types(what, x, (("dt", dt), ("B", B), ("C", C), ("z", z)), (("A", A), ("D", D), ("dt_bias", dt_bias)))
    _check_devices(what, x, (("state", state), ("dt", dt), ("A", A), ("B", B), ("C", C), ("D", D), ("z", z), ("dt_bias", dt_bias), ("slots", slots)))
    for name, t, shape in (("dt", dt, x.shape), ("z", z, x.shape), ("A", A, (channels, N)), ("C", C, B.shape), ("D", D, (channels,)),
                           ("dt_bias", dt_bias, (channels,)), ("state", state, (state.shape[0], channels, N)),
                           ("B", B, (rows, groups, N) if B.dim() == 3 else (rows, N))):
        _check_shape(what, name, t, shape)
    if state.dtype != torch.float32:
        raise TypeError(f"{what}: state must be float32, got {state.dtype}")
    _check_slots(what, rows, state, slots)
    _check_in_place(what, state)
    if _wants_grad(x, dt, A, B, C, D, z, dt_bias) or _has_tangent(state, x, dt, A, B, C, D, z, dt_bias):
        raise RuntimeError(f"{what}: a single token's step has no gradient; call it under torch.no_grad()")
    if x.device.type != "cuda":
        return baseline.naive_selective_scan_step(state, x, dt, A, B, C, D, z, dt_bias, softplus=softplus, slots=slots)
    _check_sizes(what, channels, rows)
    if B.dim() == 2:
        B, C = _grouped(B), _grouped(C)
    if torch.jit.is_tracing():
        return SelectiveScanStep.apply(state, x, dt, A, B, C, D, z, dt_bias, slots, bool(softplus))
    return _selective_step(state, x, dt, A, B, C, D, z, dt_bias, slots, softplus)


def _selective_step(state, x, dt, A, B, C, D, z, dt_bias, slots, softplus):
    L = _launching("selective_scan_step")
    with hip._on(x.device):
        x, dt, B, C, z = (_unit(t) for t in (x, dt, B, C, z))
        A, D, dt_bias, slots = (_dense(t) for t in (A, D, dt_bias, slots))
        (rows, channels), groups, N = x.shape, B.shape[1], A.shape[1]
        y = torch.empty((rows, channels), dtype=x.dtype, device=x.device)
        a = _SelectiveStep(rows, channels, groups, N, state.shape[0], _ptr(slots), int(slots is not None and slots.dtype == torch.int64),
                           _TYPES[x.dtype], int(softplus), 0, _tokens(x, 1), _tokens(dt, 1), _tokens(B, 1), _tokens(C, 1), _tokens(z, 1),
                           _tokens(y, 1), _param(A), _param(D), _param(dt_bias), state.data_ptr())
        _raise(L.scanscam_selective_step_fwd(a, _stream(x.device)), "selective_step_fwd")
    torch.autograd.graph.increment_version(state)  # (written in place)
    return y


class SelectiveScanStep(torch.autograd.Function):
    """What a trace records of a step (see ``_needs_node``); there is no gradient. A replay takes no function that is marked as changing
    its arguments, but runs functions in their order."""

    @staticmethod
    def forward(ctx, state, x, dt, A, B, C, D, z, dt_bias, slots, softplus):
        y = _selective_step(state, x, dt, A, B, C, D, z, dt_bias, slots, softplus)
        ctx.mark_non_differentiable(y)
        return y


# ------------------------------------------------------------------------------------------------------------------- convolution
def causal_conv(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None, *, activation: Optional[str] = None,
                state: Optional[torch.Tensor] = None, offsets: Optional[torch.Tensor] = None,
                return_state: bool = False) -> Union[torch.Tensor, Tuple[torch.Tensor, torch.Tensor]]:
    """
    Every channel's own causal convolution, ``y[t] = act(bias + sum_k weight[k] x[t - (K-1) + k])``.

    :param x: [batch, T, channels]
    :param weight: [channels, K], 1 to 8 taps, the last of them for the token itself; bias: [channels], optional
    :param activation: None or "silu"
    :param state: [sequences, K - 1, channels] of x's type, the inputs before the first tokens (zeros if not given)
    :param offsets: the first token of each of several packed sequences, and the end
    :param return_state: hand back the K - 1 inputs before the next token as well
    :return: y, or ``(y, state)``. Differentiable in every tensor but ``offsets``.
    """
    if _traced_through():
        if x.device.type == "cuda":
            return _eager(causal_conv, x, weight, bias, activation=activation, state=state, offsets=offsets, return_state=return_state)
    elif _native is not None:
        out = _native.conv(x, weight, bias, activation, state, offsets, return_state)
        if out is not None:
            return out
    what = "causal_conv"
    if x.dim() != 3 or weight.dim() != 2 or not 1 <= weight.shape[1] <= _MOST_TAPS:
        raise AssertionError(f"{what}: x must be [batch, T, channels] and weight [channels, 1 to {_MOST_TAPS} taps], got {tuple(x.shape)} and {tuple(weight.shape)}")
    channels, K = x.shape[2], weight.shape[1]
    _check_activation(what, activation)
    _check_types(what, x, (("state", state),), (("weight", weight), ("bias", bias)))
    _check_devices(what, x, (("weight", weight), ("bias", bias), ("state", state), ("offsets", offsets)))
    sequences = _check_offsets(what, x, offsets)
    for name, t, shape in (("weight", weight, (channels, K)), ("bias", bias, (channels,)), ("state", state, (sequences, K - 1, channels))):
        _check_shape(what, name, t, shape)
    if x.device.type != "cuda":
        return baseline.naive_causal_conv(x, weight, bias, activation=activation, state=state, offsets=offsets, return_state=return_state)
    _check_sizes(what, channels, x.shape[0] * x.shape[1], sequences)
    if _needs_node(x, weight, bias, state):
        y, new = CausalConv.apply(x, weight, bias, state, offsets, activation, bool(return_state))
    else:
        y, new, _ = _conv_forward(x, weight, bias, state, offsets, activation, return_state)
    return (y, new) if return_state else y


def _conv_args(x, weight, bias, state, offsets, activation) -> _Conv:
    a = _Conv()
    a.batch, a.T, a.channels = x.shape
    a.K, a.sequences = weight.shape[1], x.shape[0] if offsets is None else offsets.shape[0] - 1
    a.offsets, a.offsets64 = _ptr(offsets), int(offsets is not None and offsets.dtype == torch.int64)
    a.dtype, a.activation = _TYPES[x.dtype], _ACTIVATIONS[activation]
    a.x, a.weight, a.bias, a.state_in = _tokens(x), _param(weight), _param(bias), _ptr(state)
    return a


def _conv_forward(x, weight, bias, state, offsets, activation, return_state):
    L = _launching("causal_conv")
    with hip._on(x.device):
        seen = (_unit(x),) + tuple(_dense(t) for t in (weight, bias, state, offsets))
        a = _conv_args(*seen, activation)
        y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
        a.y = _tokens(y)
        new = None
        if return_state:
            new = torch.empty((a.sequences, a.K - 1, a.channels), dtype=x.dtype, device=x.device)
            a.state_out = new.data_ptr()
        _raise(L.scanscam_conv_fwd(a, _stream(x.device)), "conv_fwd")
    return y, new, seen


class CausalConv(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, state, offsets, activation, return_state):
        y, new, seen = _conv_forward(x, weight, bias, state, offsets, activation, return_state)
        ctx.save_for_backward(*seen)
        ctx.meta = _meta(*seen)
        ctx.activation = activation
        ctx.set_materialize_grads(False)
        return y, new

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, gy, gnew):
        if gy is None and gnew is None:
            return (None,) * 7
        x, *others = ctx.saved_tensors
        _check_saved("causal_conv", gy if gy is not None else gnew, dict(zip(("x", "weight", "bias", "state", "offsets"), (x, *others))), ctx.meta)
        x, (weight, bias, state, offsets) = _unit(x), (_dense(t) for t in others)  # (as above)
        L = _launching("causal_conv")
        with hip._on(x.device):
            gy = _unit(gy) if gy is not None else torch.zeros(x.shape, dtype=x.dtype, device=x.device)
            gnew = _dense(gnew)
            a = _conv_args(x, weight, bias, state, offsets, ctx.activation)
            gx = torch.empty(x.shape, dtype=x.dtype, device=x.device)
            gweight = torch.empty(weight.shape, dtype=torch.float32, device=x.device)
            gbias = None if bias is None else torch.empty(bias.shape, dtype=torch.float32, device=x.device)
            gstate = torch.empty(state.shape, dtype=x.dtype, device=x.device) if ctx.needs_input_grad[3] else None
            a.gy, a.gx = _tokens(gy), _tokens(gx)
            a.gweight, a.gbias, a.gstate_out, a.gstate_in = (_ptr(t) for t in (gweight, gbias, gnew, gstate))
            n = L.scanscam_conv_workspace_bytes(a)
            workspace = _bytes(n, x.device)
            a.workspace, a.workspace_bytes = _ptr(workspace), n
            _raise(L.scanscam_conv_bwd(a, _stream(x.device)), "conv_bwd")
            gweight = gweight.to(weight.dtype)
            return gx, gweight, None if bias is None else gbias.to(bias.dtype), gstate, None, None, None


def causal_conv_step(state: torch.Tensor, x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None, *,
                     activation: Optional[str] = None, slots: Optional[torch.Tensor] = None) -> torch.Tensor:
    """
    One token of each of several sequences: ``causal_conv``'s formula, from and into the inputs kept of each.

    :param state: [slots, K - 1, channels] of x's type, contiguous, updated in place
    :param x: [rows, channels]; weight, bias, activation as for ``causal_conv``; slots as for ``selective_scan_step``
    :return: y, [rows, channels]. Not differentiable.
    """
    if _traced_through():
        if x.device.type == "cuda":
            return _eager(causal_conv_step, state, x, weight, bias, activation=activation, slots=slots)
    elif _native is not None:
        out = _native.conv_step(state, x, weight, bias, activation, slots)
        if out is not None:
            return out
    what = "causal_conv_step"
    if x.dim() != 2 or state.dim() != 3 or weight.dim() != 2 or not 1 <= weight.shape[1] <= _MOST_TAPS:
        raise AssertionError(f"{what}: x must be [rows, channels], state [slots, K - 1, channels], weight [channels, 1 to {_MOST_TAPS} taps], "
                             f"got {tuple(x.shape)}, {tuple(state.shape)} and {tuple(weight.shape)}")
    (rows, channels), K = x.shape, weight.shape[1]
    _check_activation(what, activation)
    _check_types(what, x, (("state", state),), (("weight", weight), ("bias", bias)))
    _check_devices(what, x, (("state", state), ("weight", weight), ("bias", bias), ("slots", slots)))
    for name, t, shape in (("weight", weight, (channels, K)), ("bias", bias, (channels,)), ("state", state, (state.shape[0], K - 1, channels))):
        _check_shape(what, name, t, shape)
    _check_slots(what, rows, state, slots)
    _check_in_place(what, state)
    if _wants_grad(x, weight, bias) or _has_tangent(state, x, weight, bias):
        raise RuntimeError(f"{what}: a single token's step has no gradient; call it under torch.no_grad()")
    if x.device.type != "cuda":
        return baseline.naive_causal_conv_step(state, x, weight, bias, activation=activation, slots=slots)
    _check_sizes(what, channels, rows)
    if torch.jit.is_tracing():
        return CausalConvStep.apply(state, x, weight, bias, slots, activation)
    return _conv_step(state, x, weight, bias, slots, activation)


def _conv_step(state, x, weight, bias, slots, activation):
    L = _launching("causal_conv_step")
    with hip._on(x.device):
        x = _unit(x)
        weight, bias, slots = (_dense(t) for t in (weight, bias, slots))
        (rows, channels), K = x.shape, weight.shape[1]
        y = torch.empty((rows, channels), dtype=x.dtype, device=x.device)
        a = _ConvStep(rows, channels, K, state.shape[0], _ptr(slots), int(slots is not None and slots.dtype == torch.int64), _TYPES[x.dtype],
                      _ACTIVATIONS[activation], 0, _tokens(x, 1), _tokens(y, 1), _param(weight), _param(bias), state.data_ptr())
        _raise(L.scanscam_conv_step_fwd(a, _stream(x.device)), "conv_step_fwd")
    torch.autograd.graph.increment_version(state)
    return y


class CausalConvStep(torch.autograd.Function):
    @staticmethod
    def forward(ctx, state, x, weight, bias, slots, activation):
        y = _conv_step(state, x, weight, bias, slots, activation)
        ctx.mark_non_differentiable(y)
        return y


# -------------------------------------------------------------------------------------------------------------------------- norm
def rms_norm(x: torch.Tensor, weight: torch.Tensor, residual: Optional[torch.Tensor] = None, *, eps: float = 1e-6,
             quant: Optional[torch.dtype] = None):
    """
    Root-mean-square norm over the last dimension, with the residual's addition before it::

        sum = x + residual                     (in the residual's type; x itself without one)
        y = sum / sqrt(mean(sum^2) + eps) * weight

    What is stored in ``sum`` is what is normalised, so the gradient is that of what was computed. Squares are added up in float32: rows of values
    past some 1e19 come out as zeros.

    :param x: [..., channels], up to 32768 channels; residual: of the same shape and any supported type; weight: [channels]
    :param quant: None, ``torch.int8`` or ``torch.float8_e4m3fn``: y in 8 bits with a scale a row, ``scale = max |y| / 127`` or
        ``/ 448`` (1 for a row of zeros), y / scale rounded to nearest even
    :return: y; with a residual ``(y, sum)``; with ``quant`` ``(q, scale)`` or ``(q, scale, sum)``, scale being float32 and of x's
        leading shape. Differentiable (in x, weight and residual) unless ``quant`` is given.
    """
    if _traced_through():
        if x.device.type == "cuda":
            return _eager(rms_norm, x, weight, residual, eps=eps, quant=quant)
    elif _native is not None:
        out = _native.norm(x, weight, residual, eps, _EIGHT.get(quant, -1) if quant is not None else 0)
        if out is not None:
            return out
    what = "rms_norm"
    if x.dim() < 1 or x.shape[-1] > _MOST_NORM_CHANNELS:
        raise AssertionError(f"{what}: x must be [..., up to {_MOST_NORM_CHANNELS} channels], got shape {tuple(x.shape)}")
    _check_types(what, x, (), (("weight", weight), ("residual", residual)))
    _check_devices(what, x, (("weight", weight), ("residual", residual)))
    _check_shape(what, "weight", weight, x.shape[-1:])
    _check_shape(what, "residual", residual, x.shape)
    if quant is not None and quant not in _EIGHT:
        raise TypeError(f"{what}: quant must be None, int8 or float8_e4m3fn, got {quant}")
    if quant is not None and (_wants_grad(x, weight, residual) or _has_tangent(x, weight, residual)):
        raise RuntimeError(f"{what}: an output in 8 bits has no gradient; call it under torch.no_grad()")
    if x.device.type != "cuda":
        return baseline.naive_rms_norm(x, weight, residual, eps=eps, quant=quant)
    _check_sizes(what, x.shape[-1], x.shape[:-1].numel())
    if quant is None and _needs_node(x, weight, residual):
        y, total = RmsNorm.apply(x, weight, residual, float(eps))
        return y if residual is None else (y, total)
    if torch.jit.is_tracing():
        y, scale, total = RmsNormEight.apply(x, weight, residual, float(eps), quant)
    else:
        y, scale, total, _ = _norm_forward(x, weight, residual, eps, quant, False)
    return y if quant is None and total is None else tuple(t for t in (y, scale, total) if t is not None)


def _rows(t: Optional[torch.Tensor]) -> Optional[torch.Tensor]:
    """The tensor as rows of one stride, a view where that will do."""
    if t is None:
        return None
    t = _unit(t)
    return t.reshape(t.shape[:-1].numel(), t.shape[-1])


def _norm_args(x, weight, residual_dtype, eps) -> _Norm:
    a = _Norm()
    a.rows, a.channels = x.shape
    a.x, a.x_stride, a.weight, a.eps = x.data_ptr(), x.stride(0), _param(weight), eps
    a.dtype, a.residual_dtype = _TYPES[x.dtype], 0 if residual_dtype is None else _TYPES[residual_dtype]
    return a


def _norm_forward(x, weight, residual, eps, quant, save):
    """``(y, scale or None, sum or None, (what the backward call reads))``."""
    L = _launching("rms_norm")
    with hip._on(x.device):
        rows, more, weight = _rows(x), _rows(residual), _dense(weight)
        a = _norm_args(rows, weight, None if residual is None else residual.dtype, eps)
        y = torch.empty(x.shape, dtype=quant or x.dtype, device=x.device)
        a.y, a.out_dtype = y.data_ptr(), _EIGHT[quant] if quant is not None else a.dtype
        scale = total = rstd = None
        if residual is not None:
            total = torch.empty(x.shape, dtype=residual.dtype, device=x.device)
            a.residual, a.residual_stride, a.sum = more.data_ptr(), more.stride(0), total.data_ptr()
        if quant is not None:
            scale = torch.empty(x.shape[:-1], dtype=torch.float32, device=x.device)
            a.scale = scale.data_ptr()
        if save:
            rstd = torch.empty(rows.shape[0], dtype=torch.float32, device=x.device)
            a.rstd = rstd.data_ptr()
        _raise(L.scanscam_norm_fwd(a, _stream(x.device)), "norm_fwd")
    return y, scale, total, (rows, weight, total, rstd)


class RmsNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, residual, eps):
        y, _, total, (rows, weight, total, rstd) = _norm_forward(x, weight, residual, eps, None, True)
        kept = rows if residual is None else total, weight, rstd
        ctx.save_for_backward(*kept)
        ctx.meta = _meta(*kept)
        ctx.types = x.dtype, None if residual is None else residual.dtype
        ctx.set_materialize_grads(False)
        return y, total

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, gy, gtotal):
        kept, weight, rstd = ctx.saved_tensors
        dtype, residual_dtype = ctx.types
        shape = (gy if gy is not None else gtotal).shape if gy is not None or gtotal is not None else None
        if shape is None:
            return None, None, None, None
        _check_saved("rms_norm", gy if gy is not None else gtotal, {"rows": kept, "weight": weight, "rstd": rstd}, ctx.meta)
        L = _launching("rms_norm")
        device = kept.device
        with hip._on(device):
            gy = torch.zeros(shape, dtype=dtype, device=device) if gy is None else gy.contiguous()
            gtotal = _dense(gtotal)
            # (a hook on saved tensors may lay out what it gives back in its own way; the library takes rows of x at any distance, those of a sum dense)
            rows, weight, rstd = _rows(kept if residual_dtype is None else kept.contiguous()), _dense(weight), _dense(rstd)
            a = _norm_args(rows, weight, residual_dtype, 0.0)
            a.dtype, a.rstd, a.gy, a.gsum = _TYPES[dtype], rstd.data_ptr(), gy.data_ptr(), _ptr(gtotal)
            gx = torch.empty(shape, dtype=dtype, device=device)
            gresidual = None
            if residual_dtype is not None:
                a.residual, a.sum = rows.data_ptr(), rows.data_ptr()
                # (where the types agree the two gradients are the same values)
                gresidual = gx if residual_dtype == dtype else torch.empty(shape, dtype=residual_dtype, device=device)
            gweight = torch.empty(weight.shape, dtype=torch.float32, device=device)
            a.gx, a.gresidual, a.gweight = gx.data_ptr(), None if gresidual is None or gresidual is gx else gresidual.data_ptr(), gweight.data_ptr()
            n = L.scanscam_norm_workspace_bytes(a)
            workspace = _bytes(n, device)
            a.workspace, a.workspace_bytes = _ptr(workspace), n
            _raise(L.scanscam_norm_bwd(a, _stream(device)), "norm_bwd")
            return gx, gweight.to(weight.dtype), gresidual, None


class RmsNormEight(torch.autograd.Function):
    """What a trace records of a norm in 8 bits; there is no gradient."""

    @staticmethod
    def forward(ctx, x, weight, residual, eps, quant):
        y, scale, total, _ = _norm_forward(x, weight, residual, eps, quant, False)
        ctx.mark_non_differentiable(*(t for t in (y, scale, total) if t is not None))
        return y, scale, total
