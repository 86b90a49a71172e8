"""
Calls of the state space layer's operators that are not plain ones: forward-mode derivatives, recorded calls. None of them may give
an answer that looks right and is not.
"""
import pytest
import torch
from torch.autograd import forward_ad

import scanscam_amd as f
from scanscam_amd import state_space

pytestmark = pytest.mark.gpu


def calls(gpu, seed=0):
    """name: (function of tensors, the tensors), without gradients of their own."""
    g = torch.Generator(device=gpu).manual_seed(seed)
    r = lambda *s: torch.randn(s, generator=g, device=gpu)  # noqa: E731
    x, dt, z, B, C = r(2, 37, 24), r(2, 37, 24), r(2, 37, 24), r(2, 37, 2, 8), r(2, 37, 2, 8)
    A, D, bias, state, w, kept = -r(24, 8).exp(), r(24), r(24), r(2, 24, 8), r(24, 4), r(2, 3, 24)
    return {
        "rms_norm": (lambda x, w: f.rms_norm(x, w), (x, D)),
        "rms_norm_residual": (lambda x, w, r: f.rms_norm(x, w, r), (x, D, z)),
        "causal_conv": (lambda x, w, b: f.causal_conv(x, w, b, activation="silu"), (x, w, bias)),
        "causal_conv_state": (lambda x, w, b, s: f.causal_conv(x, w, b, state=s, return_state=True), (x, w, bias, kept)),
        "selective_scan": (lambda *t: f.selective_scan(*t, softplus=True), (x, dt, A, B, C, D, z, bias)),
        "selective_scan_state": (lambda s, *t: f.selective_scan(*t, state=s, return_state=True), (state, x, dt.abs(), A, B, C)),
    }


def single(gpu, seed=0):
    """The calls that have no gradient, the steps with their state first."""
    g = torch.Generator(device=gpu).manual_seed(seed)
    r = lambda *s: torch.randn(s, generator=g, device=gpu)  # noqa: E731
    slots = torch.tensor([4, 0, -1, 2], device=gpu)
    return {
        "rms_norm_int8": (lambda x, w: f.rms_norm(x, w, quant=torch.int8), (r(5, 40), r(40))),
        "rms_norm_int8_residual": (lambda x, w, s: f.rms_norm(x, w, s, quant=torch.int8), (r(5, 40), r(40), r(5, 40))),
        "selective_scan_step": (lambda s, *t: f.selective_scan_step(s, *t, softplus=True, slots=slots), (r(6, 24, 8), r(4, 24), r(4, 24), -r(24, 8).exp(), r(4, 8), r(4, 8))),
        "causal_conv_step": (lambda s, *t: f.causal_conv_step(s, *t, activation="silu", slots=slots), (r(6, 3, 24), r(4, 24), r(24, 4), r(24))),
    }


def listed(out):
    return list(out) if isinstance(out, (tuple, list)) else [out]


@pytest.mark.parametrize("name", list(calls("cpu")) + list(single("cpu")))
def test_forward_mode_is_refused(gpu, name):
    """As scan() refuses it; an output without a tangent would be a derivative of zero."""
    fn, tensors = {**calls(gpu), **single(gpu)}[name]
    for i in range(len(tensors)):
        for grads in (True, False):
            with forward_ad.dual_level(), torch.set_grad_enabled(grads):
                dual = [forward_ad.make_dual(t, torch.ones_like(t)) if k == i else t for k, t in enumerate(tensors)]
                with pytest.raises(RuntimeError):  # (NotImplementedError is one)
                    fn(*dual)
    with forward_ad.dual_level():  # nothing of the call's has a tangent
        assert all(torch.isfinite(o.float()).all() for o in listed(fn(*[t.clone() for t in tensors])))


@pytest.mark.parametrize("name", list(calls("cpu")) + list(single("cpu")))
def test_a_trace_runs_the_kernels(gpu, name):
    """A call that torch.jit.trace recorded computes when it is replayed, with other inputs than those it saw, and updates states in place."""
    fn, tensors = {**calls(gpu), **single(gpu)}[name]
    with torch.no_grad():
        traced = torch.jit.trace(fn, [t.clone() for t in tensors], check_trace=False)
        for seed in (1, 2):
            given = {**calls(gpu, seed), **single(gpu, seed)}[name][1]
            outs = []
            for call in (fn, traced):
                for n in (1 << 16, 1 << 10):
                    torch.full((n,), float("nan"), device=gpu)  # (memory that an output which nothing writes would show)
                own = [t.clone() for t in given]
                outs.append([*listed(call(*own)), *own])
            assert len(outs[0]) == len(outs[1]) and all(torch.equal(p, q) for p, q in zip(*outs))
    if name in calls("cpu"):  # recorded without gradients, replayed with them
        grads = []
        for call in (fn, traced):
            leaves = [t.clone().requires_grad_() for t in tensors]
            grads.append(torch.autograd.grad([o.square().sum() for o in listed(call(*leaves))], leaves))
        assert all(torch.equal(p, q) for p, q in zip(*grads))


def test_a_trace_of_several_steps_takes_them_in_order(gpu):
    (scan, state, *t), (conv, kept, *u) = ((fn, *given) for fn, given in (single(gpu)[n] for n in ("selective_scan_step", "causal_conv_step")))

    def three(state, kept, x, *rest):
        outs = []
        for _ in range(3):
            x = scan(state, conv(kept, x, *u[1:]), *t[1:])
            outs += [x, state.sum()]
        return tuple(outs)

    with torch.no_grad():
        traced = torch.jit.trace(three, (state.clone(), kept.clone(), t[0]), check_trace=False)
        for scale in (1.0, 0.5):
            outs = []
            for call in (three, traced):
                own = [state.clone(), kept.clone(), t[0] * scale]
                outs.append([*call(*own), *own])
            assert all(torch.equal(p, q) for p, q in zip(*outs))


@pytest.mark.parametrize("name", list(calls("cpu")) + list(single("cpu")))
def test_make_fx_is_refused(gpu, name):
    """It records ATen calls, of which these are none; its graph would return outputs that nothing writes. (CPU tensors' calls are.)"""
    from torch.fx.experimental.proxy_tensor import make_fx

    fn, tensors = {**calls(gpu), **single(gpu)}[name]
    for mode in ("real", "fake"):
        with torch.no_grad(), pytest.raises(RuntimeError, match="make_fx"):
            make_fx(fn, tracing_mode=mode)(*tensors)
    if name in single("cpu"):
        return

    def gradients(*t):
        leaves = [v.detach().requires_grad_() for v in t]
        return torch.autograd.grad([o.sum() for o in listed(fn(*leaves))], leaves)

    with pytest.raises(RuntimeError, match="make_fx"):
        make_fx(gradients)(*tensors)
    leaves = [t.clone().requires_grad_() for t in tensors]
    outs = listed(fn(*leaves))
    with pytest.raises(RuntimeError, match="make_fx"):  # the backward pass of a call made outside
        make_fx(lambda *g: torch.autograd.grad(outs, leaves, g))(*[torch.ones_like(o) for o in outs])


@pytest.mark.parametrize("backend", ["eager", "aot_eager"])
def test_calls_from_compiled_functions(gpu, backend):
    """torch.compile breaks its graph at a call, which then is what it is elsewhere, as scan()'s calls are."""
    for name, (fn, tensors) in {**calls(gpu), **single(gpu)}.items():
        def user(first, *rest):
            return [o.float() * 2 for o in listed(fn(first, *rest))]

        for grad in (False, True) if name in calls("cpu") else (False,):
            torch._dynamo.reset()
            results = []
            for call in (user, torch.compile(user, backend=backend)):
                own = [t.clone().requires_grad_(grad) for t in tensors]
                outs = call(*own)
                results.append(outs + (list(torch.autograd.grad([o.sum() for o in outs], own)) if grad else own))
            assert all(torch.equal(p, q) for p, q in zip(*results)), (name, grad)
    torch._dynamo.reset()


def test_a_backward_pass_that_is_compiled(gpu):
    """Compiled autograd calls the native nodes as they are."""
    from torch._dynamo import compiled_autograd

    for name, (fn, tensors) in calls(gpu).items():
        grads = []
        for compiled in (False, True):
            torch._dynamo.reset()
            leaves = [t.clone().requires_grad_() for t in tensors]
            loss = sum(o.square().sum() for o in listed(fn(*leaves)))
            if compiled:
                with compiled_autograd._enable(torch.compile(backend="eager")):
                    loss.backward()
            else:
                loss.backward()
            grads.append([t.grad for t in leaves])
        assert all(torch.equal(p, q) for p, q in zip(*grads)), name
    torch._dynamo.reset()


def rows_apart(t):
    """The same values, unit-stride at the end, rows further apart than they are long."""
    if t.dim() < 2:
        return t
    out = torch.full((*t.shape[:-1], 2, t.shape[-1]), float("nan"), dtype=t.dtype, device=t.device)[..., 0, :]
    return out.copy_(t)


def one_row(t):
    """The same values, where all rows are alike, as one row at a distance of zero."""
    return t if t.dim() < 2 else t[(slice(0, 1),) * (t.dim() - 1)].expand(t.shape)


@pytest.mark.parametrize("native", [True, False])
@pytest.mark.parametrize("residual", [None, torch.float32, torch.bfloat16])
@pytest.mark.parametrize("unpack", [rows_apart, one_row])
def test_norm_of_saved_rows_at_other_strides(gpu, monkeypatch, native, residual, unpack):
    """What hooks on saved tensors give back may lie elsewhere in memory in a layout of its own: the gradients are the same bits."""
    if not native:
        monkeypatch.setattr(state_space, "_native", None)
    g = torch.Generator(device=gpu).manual_seed(3)
    row = torch.randn(1, 1, 40, generator=g, device=gpu)
    x = row.expand(3, 7, 40).contiguous() if unpack is one_row else torch.randn(3, 7, 40, generator=g, device=gpu)
    x, w, gy = x.to(torch.bfloat16), torch.randn(40, generator=g, device=gpu), torch.randn(3, 7, 40, generator=g, device=gpu).to(torch.bfloat16)
    r = None if residual is None else (x * 3).to(residual)
    grads = []
    for give in (lambda t: t, unpack):
        leaves = [t.clone().requires_grad_() for t in (x, w, r) if t is not None]
        with torch.autograd.graph.saved_tensors_hooks(lambda t: t.detach(), give):
            out = f.rms_norm(*leaves)
        grads.append(torch.autograd.grad(out if residual is None else out[0], leaves, gy))
    assert all(torch.equal(p, q) for p, q in zip(*grads))


@pytest.mark.parametrize("native", [True, False])
@pytest.mark.parametrize("changed", ["device", "type", "shape"])
def test_saved_tensors_that_hooks_changed_are_refused(gpu, monkeypatch, native, changed):
    """A hook on saved tensors that gives back another device's memory, another type or fewer values: an error, for each of the saved ones."""
    if not native:
        monkeypatch.setattr(state_space, "_native", None)
    give = {"device": lambda t: t.cpu(), "type": lambda t: t.double(), "shape": lambda t: t[:-1]}[changed]
    g = torch.Generator(device=gpu).manual_seed(7)
    r = lambda *s: torch.randn(s, generator=g, device=gpu)  # noqa: E731
    offsets = torch.tensor([0, 30, 30, 70], dtype=torch.int32, device=gpu)
    cases = {
        "rms_norm": lambda p: f.rms_norm(r(4, 9, 40).requires_grad_(), p(40)),
        "rms_norm_residual": lambda p: f.rms_norm(r(4, 9, 40).requires_grad_(), p(40), r(4, 9, 40)),
        "causal_conv": lambda p: f.causal_conv(r(1, 70, 24).requires_grad_(), p(24, 4), p(24), state=r(3, 3, 24), offsets=offsets, return_state=True),
        "selective_scan": lambda p: f.selective_scan(r(1, 70, 24).requires_grad_(), r(1, 70, 24), p(24, 8) - 3, r(1, 70, 2, 8), r(1, 70, 2, 8), p(24), r(1, 70, 24), p(24),
                                                     softplus=True, state=r(3, 24, 8), offsets=offsets, return_state=True),
    }
    for name, call in cases.items():
        seen = []

        def pack(t):
            seen.append(t)
            return len(seen) - 1

        with torch.autograd.graph.saved_tensors_hooks(pack, lambda i: seen[i].clone()):
            call(lambda *s: r(*s).requires_grad_())
        count = len(seen)
        assert count >= 3
        for k in range(count):
            seen.clear()
            own = []
            with torch.autograd.graph.saved_tensors_hooks(pack, lambda i: give(seen[i]) if i == k else seen[i].clone()):
                outs = listed(call(lambda *s: own.append(r(*s).requires_grad_()) or own[-1]))
            for which in range(len(outs)):  # the gradient of one output or the other
                print(name, changed, native, "saved tensor", k, tuple(seen[k].shape), "output", which, flush=True)
                with pytest.raises(RuntimeError, match="saved for the backward pass"):
                    torch.autograd.grad(outs[which].sum(), own, retain_graph=True)
