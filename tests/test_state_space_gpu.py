"""
The state space layer's kernels against the plain loops of scanscam_amd.baseline in float64 on the same stored inputs, gradients
against those that torch.autograd takes of these loops and against differences.

Bound of every comparison: half a unit in the last place of the output's type (half of its epsilon, of the value), plus
(64 + 2 T) roundings of 2^-24 at the size of the tensor's largest value: a value that goes through a recurrence of T steps is
rounded at most twice a step (the decay's product and the sum, both relative to a state that the decays only shrink), and
some 64 times outside of it (exponentials, softplus, gates, sums over states, channels and tokens, which are taken in short chains).
"""
import pytest
import torch

import scanscam_amd as f
from scanscam_amd import baseline, state_space

pytestmark = pytest.mark.gpu

HALF = {t: torch.finfo(t).eps / 2 for t in (torch.float32, torch.bfloat16, torch.float16)}


def close(got, want, T, what):
    assert got.shape == want.shape, (what, got.shape, want.shape)
    if got.numel() == 0:
        return
    got, half = got.detach().cpu(), HALF[got.dtype]
    got, want = got.double(), want.detach().double()
    bound = half * 1.01 * want.abs() + (64 + 2 * T) * 2.0 ** -24 * want.abs().max()
    if half > 2.0 ** -24:  # the smallest numbers of fp16 are further apart than its relative precision
        bound = bound + 2.0 ** -25
    over = (got - want).abs() - bound
    assert torch.isfinite(got).all() and (over <= 0).all(), f"{what}: {float((got - want).abs().max()):.3e} off, bound {float(bound.min()):.3e}"


def offsets_of(lengths, dtype=torch.int32):
    return torch.tensor([0] + torch.tensor(lengths).cumsum(0).tolist(), dtype=dtype)


def make_scan(seed, dtype, batch, T, D, N, groups=1, z=True, skip=True, bias=True, lengths=None, state=False, param=torch.float32):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(s, generator=g)  # noqa: E731
    if lengths is not None:
        batch, T = 1, sum(lengths)
    v = {"x": r(batch, T, D), "dt": r(batch, T, D) * 0.5, "A": -torch.arange(1.0, N + 1) * (r(D, N) * 0.2).exp(), "B": r(batch, T, groups, N), "C": r(batch, T, groups, N)}
    v = {k: t.to(param if k == "A" else dtype) for k, t in v.items()}
    v["D"] = r(D).to(param) if skip else None
    v["z"] = r(batch, T, D).to(dtype) if z else None
    v["dt_bias"] = (r(D) - 3).to(param) if bias else None
    sequences = batch if lengths is None else len(lengths)
    v["state"] = r(sequences, D, N) if state else None
    v["offsets"] = offsets_of(lengths) if lengths is not None else None
    return v


def wide(t):
    return t if t is None or not t.is_floating_point() else t.double()


SCANS = [
    # dtype, batch, T, D, N, and what differs
    (torch.float32, 2, 300, 40, 16, {}),
    (torch.float32, 1, 1, 1, 1, {}),
    (torch.float32, 3, 0, 8, 4, {"state": True}),
    (torch.float32, 2, 127, 33, 3, {"z": False, "state": True}),
    (torch.float32, 1, 128, 64, 17, {"skip": False}),
    (torch.float32, 1, 129, 5, 40, {"bias": False, "groups": 5, "state": True}),
    (torch.float32, 2, 9, 96, 16, {"groups": 2, "state": True}),
    (torch.float32, 1, 260, 6, 256, {}),
    (torch.float32, 0, 0, 30, 8, {"lengths": [1, 0, 130, 0, 0, 64, 257, 0], "state": True}),
    (torch.float32, 0, 0, 70, 16, {"lengths": [0, 3, 8, 1], "z": False}),
    (torch.bfloat16, 2, 200, 100, 16, {"groups": 4, "state": True}),
    (torch.bfloat16, 0, 0, 64, 16, {"lengths": [128, 5, 0, 300], "state": True}),
    (torch.bfloat16, 1, 33, 31, 8, {"param": torch.bfloat16}),
    (torch.float16, 2, 140, 48, 16, {"param": torch.float16}),
    (torch.float32, 1, 1500, 9, 16, {"state": True}),
]


@pytest.mark.parametrize("dtype,batch,T,D,N,more", SCANS, ids=lambda v: str(v).replace("torch.", "").replace(" ", ""))
@pytest.mark.parametrize("softplus,parts", [(True, 0), (False, 0), (True, 2), (True, 5)])
def test_scan_and_gradients(gpu, monkeypatch, dtype, batch, T, D, N, more, softplus, parts):
    monkeypatch.setattr(state_space, "_parts", parts)  # parts of time to share out, also where there is less than a tile for each
    v = make_scan(5, dtype, batch, T, D, N, **more)
    if not softplus:  # step sizes themselves
        v["dt"] = (v["dt"].float().abs() * 0.2).to(dtype)
        v["dt_bias"] = None if v["dt_bias"] is None else (v["dt_bias"].float().abs() * 0.01).to(v["dt_bias"].dtype)
    state = v["state"] is not None
    grad_of = [k for k, t in v.items() if t is not None and k != "offsets"]
    ref = {k: wide(t).requires_grad_() if k in grad_of else t for k, t in v.items()}
    want, want_state = baseline.naive_selective_scan(**ref, softplus=softplus, return_state=True)
    g = torch.Generator().manual_seed(6)
    gy, gs = torch.randn(want.shape, generator=g).to(dtype), torch.randn(want_state.shape, generator=g)
    outs, weights = (want, want_state) if state else (want,), (gy.double(), gs.double()) if state else (gy.double(),)
    want_grads = torch.autograd.grad(outs, [ref[k] for k in grad_of], weights, allow_unused=True)

    dev = {k: None if t is None else t.to(gpu).requires_grad_(k in grad_of) for k, t in v.items()}
    with torch.no_grad():
        plain = f.selective_scan(**dev, softplus=softplus)
    got = f.selective_scan(**dev, softplus=softplus, return_state=state)
    got, got_state = got if state else (got, None)
    assert torch.equal(plain, got.detach())
    Tn = v["x"].shape[1]
    close(got, want, Tn, "y")
    if state:
        close(got_state, want_state, Tn, "state")
    outs, weights = ((got, got_state), (gy.to(gpu), gs.to(gpu))) if state else ((got,), (gy.to(gpu),))
    grads = torch.autograd.grad(outs, [dev[k] for k in grad_of], weights)
    again = torch.autograd.grad(f.selective_scan(**dev, softplus=softplus, return_state=state) if state else (f.selective_scan(**dev, softplus=softplus),),
                                [dev[k] for k in grad_of], weights)
    for k, a, b, w in zip(grad_of, grads, again, want_grads):
        assert a.dtype == v[k].dtype and torch.equal(a, b), k  # (the order of every sum is fixed)
        close(a, torch.zeros(v[k].shape, dtype=torch.float64) if w is None else w, Tn, f"gradient of {k}")


@pytest.mark.parametrize("dtype,batch,T,D,N,more", [(torch.float32, 2, 140, 8190, 16, {}), (torch.bfloat16, 64, 9, 255, 5, {"state": True}),
                                                     (torch.float32, 0, 0, 64, 16, {"lengths": [3, 0, 1, 7] * 66})],
                         ids=lambda v: str(v).replace("torch.", "").replace(" ", "")[:30])
def test_scan_of_many_channels(gpu, monkeypatch, dtype, batch, T, D, N, more):
    """Enough workgroups for the backward kernel to take two sets of channels each."""
    test_scan_and_gradients(gpu, monkeypatch, dtype, batch, T, D, N, more, True, 0)


def test_scan_of_projections_parts(gpu):
    """Views of wider projections, odd offsets, broadcast inputs and other orders of dimensions give what dense tensors give."""
    v = make_scan(11, torch.bfloat16, 2, 70, 24, 8)
    d = {k: None if t is None else t.to(gpu) for k, t in v.items()}
    want = f.selective_scan(**d, softplus=True)
    xz = torch.zeros(2, 70, 51, dtype=torch.bfloat16, device=gpu)
    xz[..., 1:25], xz[..., 27:51] = d["x"], d["z"]
    parts = torch.zeros(2, 70, 19, dtype=torch.bfloat16, device=gpu)
    parts[..., 3:11], parts[..., 11:19] = d["B"][:, :, 0], d["C"][:, :, 0]
    other = dict(d, x=xz[..., 1:25], z=xz[..., 27:51], B=parts[..., 3:11], C=parts[..., 11:19], dt=d["dt"].permute(2, 0, 1).contiguous().permute(1, 2, 0),
                 A=d["A"].t().contiguous().t())
    assert torch.equal(f.selective_scan(**other, softplus=True), want)
    one = d["x"][:1, :1].expand(2, 70, 24)
    assert torch.equal(f.selective_scan(**dict(d, x=one), softplus=True), f.selective_scan(**dict(d, x=one.contiguous()), softplus=True))
    # a gradient that is a broadcast, as that of sum() is
    leaf = {k: None if t is None else t.clone().requires_grad_() for k, t in d.items()}
    y = f.selective_scan(**leaf, softplus=True)
    a = torch.autograd.grad(y, leaf["dt"], torch.ones((), dtype=y.dtype, device=gpu).expand(y.shape), retain_graph=True)[0]
    assert torch.equal(a, torch.autograd.grad(y, leaf["dt"], torch.ones_like(y))[0])


@pytest.mark.parametrize("cut", [1, 64, 128, 200])
def test_scan_in_pieces(gpu, cut):
    """The state handed on from one call to the next, and single tokens after that, continue the sequence."""
    v = make_scan(3, torch.float32, 2, 260, 40, 16)
    d = {k: None if t is None else t.to(gpu) for k, t in v.items()}
    want, want_state = baseline.naive_selective_scan(**{k: wide(t) for k, t in v.items()}, softplus=True, return_state=True)
    seqs = ("x", "dt", "B", "C", "z")
    part = lambda a, b: {k: t[:, a:b] if k in seqs else t for k, t in d.items()}  # noqa: E731
    y0, state = f.selective_scan(**part(0, cut), softplus=True, return_state=True)
    y1, state = f.selective_scan(**dict(part(cut, 255), state=state), softplus=True, return_state=True)
    rest = []
    for t in range(255, 260):
        token = {k: d[k][:, t] for k in seqs}
        rest.append(f.selective_scan_step(state, token["x"], token["dt"], d["A"], token["B"], token["C"], d["D"], token["z"], d["dt_bias"], softplus=True))
    close(torch.cat((y0, y1, torch.stack(rest, 1)), 1), want, 260, "y")
    close(state, want_state, 260, "state")


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows,D,N,groups", [(1, 1, 1, 1), (3, 65, 16, 1), (5, 40, 5, 2), (2, 24, 64, 3), (2, 7, 130, 7), (2, 100, 256, 1), (70, 33, 8, 1)])
@pytest.mark.parametrize("wide_slots", [True, False])
def test_scan_step(gpu, dtype, rows, D, N, groups, wide_slots):
    v = make_scan(8, dtype, rows, 1, D, N, groups)
    slots = torch.randperm(rows + 4, generator=torch.Generator().manual_seed(1))[:rows]
    if rows > 2:
        slots[1], slots[2] = -1, rows + 4  # rows without a sequence
    slots = slots.to(torch.int64 if wide_slots else torch.int32)
    state = torch.randn(rows + 4, D, N, generator=torch.Generator().manual_seed(2))
    args = [None if v[k] is None else v[k][:, 0] if k in ("x", "dt", "B", "C", "z") else v[k] for k in ("x", "dt", "A", "B", "C", "D", "z", "dt_bias")]
    want_state = state.double()
    want = baseline.naive_selective_scan_step(want_state, *[wide(t) for t in args], softplus=True, slots=slots)
    dev = state.to(gpu)
    got = f.selective_scan_step(dev, *[None if t is None else t.to(gpu) for t in args], softplus=True, slots=slots.to(gpu))
    close(got, want, 1, "y")
    close(dev, want_state, 1, "state")
    untouched = [s for s in range(rows + 4) if s not in slots.tolist()]
    assert torch.equal(dev[untouched].cpu(), state[untouched])


def test_scan_extremes(gpu):
    """Large step sizes forget everything, zero ones nothing, and one channel's infinity stays in its channel and sequence."""
    v = make_scan(4, torch.float32, 1, 0, 8, 16, lengths=[200, 150], bias=False, z=False)
    v["dt"][:, 100] = 200.0
    v["dt"][:, 120:140] = -200.0
    want, state = baseline.naive_selective_scan(**{k: wide(t) for k, t in v.items()}, softplus=True, return_state=True)
    d = {k: None if t is None else t.to(gpu) for k, t in v.items()}
    got, got_state = f.selective_scan(**d, softplus=True, return_state=True)
    close(got, want, 350, "y")
    close(got_state, state, 350, "state")
    for bad in (float("inf"), float("nan")):
        x = d["x"].clone()
        x[0, 50, 3] = bad
        y = f.selective_scan(**dict(d, x=x), softplus=True)
        same = torch.ones_like(y, dtype=torch.bool)
        same[0, 50:200, 3] = False
        assert torch.equal(y[same], got[same]) and not torch.isfinite(y[0, 50:200, 3]).any()


def test_scan_gradient_against_differences(gpu):
    """The change of a weighted sum of the outputs along a random direction. In float32 a difference over steps of 2 h = 2^-5 has an error of
    h^2 / 6 times the third derivative (the direction is scaled so that nothing changes by more than some per cent) and of
    2^-24 sqrt(values) / h from rounding; 2 % of the sum's change covers both."""
    v = make_scan(9, torch.float32, 2, 150, 24, 16, groups=2, state=True)
    d = {k: None if t is None else t.to(gpu).requires_grad_() for k, t in v.items()}
    y, s = f.selective_scan(**d, softplus=True, return_state=True)
    gen = torch.Generator().manual_seed(3)
    wy, ws = torch.randn(y.shape, generator=gen).to(gpu), torch.randn(s.shape, generator=gen).to(gpu)
    names = [k for k in d if d[k] is not None]
    grads = dict(zip(names, torch.autograd.grad((y, s), [d[k] for k in names], (wy, ws))))
    for k in names:
        along = grads[k].sign() * torch.rand(v[k].shape, generator=gen).to(gpu)
        if k == "A":
            along = along * d[k].detach().abs()
        h = 2.0 ** -6

        def value(sign):
            moved = {n: None if t is None else (t.detach() + sign * h * along if n == k else t.detach()) for n, t in d.items()}
            y, s = f.selective_scan(**moved, softplus=True, return_state=True)
            return float((y.double() * wy.double()).sum() + (s.double() * ws.double()).sum())

        slope, want = (value(1) - value(-1)) / (2 * h), float((grads[k].double() * along.double()).sum())
        assert abs(slope - want) <= 0.02 * abs(want), (k, slope, want)


CONVS = [
    (torch.float32, 2, 100, 40, 4, {}),
    (torch.float32, 1, 1, 1, 1, {}),
    (torch.float32, 2, 2, 5, 8, {"state": True}),
    (torch.float32, 3, 0, 4, 3, {"state": True}),
    (torch.float32, 2, 131, 33, 3, {"bias": False, "state": True}),
    (torch.float32, 0, 0, 20, 4, {"lengths": [1, 0, 70, 0, 0, 2, 129, 3, 0], "state": True}),
    (torch.bfloat16, 2, 257, 72, 4, {"state": True}),
    (torch.bfloat16, 0, 0, 65, 2, {"lengths": [0, 64, 1, 200]}),
    (torch.bfloat16, 1, 50, 7, 5, {"param": torch.bfloat16}),
    (torch.float16, 2, 90, 64, 6, {"param": torch.float16, "state": True}),
    (torch.float16, 2, 40, 24, 7, {}),
]


@pytest.mark.parametrize("dtype,batch,T,D,K,more", CONVS, ids=lambda v: str(v).replace("torch.", "").replace(" ", ""))
@pytest.mark.parametrize("activation", [None, "silu"])
def test_conv_and_gradients(gpu, dtype, batch, T, D, K, more, activation):
    g = torch.Generator().manual_seed(21)
    lengths, param, state = more.get("lengths"), more.get("param", torch.float32), more.get("state", False)
    if lengths is not None:
        batch, T = 1, sum(lengths)
    v = {"x": torch.randn(batch, T, D, generator=g).to(dtype), "weight": torch.randn(D, K, generator=g).to(param),
         "bias": torch.randn(D, generator=g).to(param) if more.get("bias", True) else None,
         "state": torch.randn(batch if lengths is None else len(lengths), K - 1, D, generator=g).to(dtype) if state else None}
    offsets = offsets_of(lengths, torch.int64) if lengths is not None else None
    names = [k for k in v if v[k] is not None]
    ref = {k: None if t is None else t.double().requires_grad_() for k, t in v.items()}
    want, want_state = baseline.naive_causal_conv(**ref, activation=activation, offsets=offsets, return_state=True)
    gy, gs = torch.randn(want.shape, generator=g).to(dtype), torch.randn(want_state.shape, generator=g).to(dtype)
    dev = {k: None if t is None else t.to(gpu).requires_grad_() for k, t in v.items()}
    off = None if offsets is None else offsets.to(gpu)
    got, got_state = f.causal_conv(**dev, activation=activation, offsets=off, return_state=True)
    close(got, want, 1, "y")
    assert torch.equal(got_state.detach().cpu().double(), want_state.detach())
    want_grads = torch.autograd.grad((want, want_state), [ref[k] for k in names], (gy.double(), gs.double()), allow_unused=True)
    grads = torch.autograd.grad((got, got_state), [dev[k] for k in names], (gy.to(gpu), gs.to(gpu)))
    for k, a, w in zip(names, grads, want_grads):
        assert a.dtype == v[k].dtype
        close(a, torch.zeros(v[k].shape, dtype=torch.float64) if w is None else w, T // 8, f"gradient of {k}")
    only = torch.autograd.grad(f.causal_conv(**dev, activation=activation, offsets=off), [dev[k] for k in names], gy.to(gpu))
    want_only = torch.autograd.grad(baseline.naive_causal_conv(**ref, activation=activation, offsets=offsets), [ref[k] for k in names], gy.double(), allow_unused=True) if T else [None] * len(names)
    for k, a, w in zip(names, only, want_only):
        close(a, torch.zeros(v[k].shape, dtype=torch.float64) if w is None else w, T // 8, f"gradient of {k}")


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows,D,K", [(1, 1, 1), (4, 65, 4), (3, 24, 8), (70, 9, 2)])
def test_conv_step(gpu, dtype, rows, D, K):
    g = torch.Generator().manual_seed(31)
    x, w, b = torch.randn(rows, 2 * D, generator=g).to(dtype)[:, D:], torch.randn(D, K, generator=g), torch.randn(D, generator=g)
    state = torch.randn(rows + 2, K - 1, D, generator=g).to(dtype)
    slots = torch.randperm(rows + 2, generator=g)[:rows].to(torch.int32)
    if rows > 3:
        slots[2], slots[0] = -7, rows + 2
    want_state = state.double()
    want = baseline.naive_causal_conv_step(want_state, x.double(), w.double(), b.double(), activation="silu", slots=slots)
    dev = state.to(gpu)
    got = f.causal_conv_step(dev, x.to(gpu), w.to(gpu), b.to(gpu), activation="silu", slots=slots.to(gpu))
    close(got, want, 1, "y")
    assert torch.equal(dev.cpu().double(), want_state)


def test_conv_continues_with_single_tokens(gpu):
    g = torch.Generator().manual_seed(33)
    x, w = torch.randn(2, 80, 24, generator=g), torch.randn(24, 4, generator=g)
    want = baseline.naive_causal_conv(x.double(), w.double())
    d, dw = x.to(gpu), w.to(gpu)
    y0, state = f.causal_conv(d[:, :2], dw, return_state=True)  # fewer tokens than the state has rows
    y1, state = f.causal_conv(d[:, 2:70], dw, state=state, return_state=True)
    rest = [f.causal_conv_step(state, d[:, t], dw) for t in range(70, 80)]
    close(torch.cat((y0, y1, torch.stack(rest, 1)), 1), want, 1, "y")


NORMS = [
    (torch.float32, None, (3, 5, 64)), (torch.float32, torch.float32, (7, 1)), (torch.float32, torch.bfloat16, (2, 2049)), (torch.float32, None, (0, 16)),
    (torch.bfloat16, None, (65, 1000)), (torch.bfloat16, torch.bfloat16, (4, 2, 2048)), (torch.bfloat16, torch.float32, (9, 4096)),
    (torch.bfloat16, torch.float32, (3, 5000)), (torch.float16, torch.float16, (5, 9001)), (torch.float16, torch.float32, (2, 32768)),
    (torch.bfloat16, torch.float32, (3000, 40)), (torch.float16, None, (33,)), (torch.bfloat16, torch.float32, (5, 32767)), (torch.bfloat16, None, (4, 32763)),
    (torch.bfloat16, torch.bfloat16, (1100, 2047)), (torch.float32, None, (1030, 513)), (torch.bfloat16, torch.float32, (1024, 2560)),
]


@pytest.mark.parametrize("dtype,residual,shape", NORMS, ids=lambda v: str(v).replace("torch.", "").replace(" ", ""))
@pytest.mark.parametrize("param", [torch.float32, torch.bfloat16])
def test_norm_and_gradients(gpu, dtype, residual, shape, param):
    g = torch.Generator().manual_seed(41)
    v = {"x": torch.randn(shape, generator=g).to(dtype), "weight": (1 + 0.2 * torch.randn(shape[-1], generator=g)).to(param)}
    total = v["x"]
    if residual is not None:
        v["residual"] = (2 * torch.randn(shape, generator=g)).to(residual)
        total = (v["x"].float() + v["residual"].float()).to(residual)  # what is stored is what is normalised
    dev = {k: t.to(gpu).requires_grad_() for k, t in v.items()}
    got = f.rms_norm(**dev, eps=1e-5)
    if residual is not None:
        got, got_total = got
        assert got_total.dtype == residual and torch.equal(got_total.cpu(), total)
    r, w = total.double().requires_grad_(), v["weight"].double().requires_grad_()
    want = r / torch.sqrt(r.square().mean(-1, keepdim=True) + 1e-5) * w
    assert got.dtype == dtype
    close(got, want, 0, "y")
    gy, gt = torch.randn(shape, generator=g).to(dtype), torch.randn(shape, generator=g).to(total.dtype)
    gr, gw = torch.autograd.grad(want, (r, w), gy.double())
    both = residual is not None
    grads = dict(zip(v, torch.autograd.grad((got, got_total) if both else got, list(dev.values()), (gy.to(gpu), gt.to(gpu)) if both else gy.to(gpu))))
    rows = v["x"].numel() // shape[-1]
    close(grads["weight"], gw, rows // 64, "gradient of weight")
    if both:
        gr = gr + gt.double()
        close(grads["residual"], gr, 0, "gradient of residual")
    close(grads["x"], gr, 0, "gradient of x")


@pytest.mark.parametrize("quant,limit", [(torch.int8, 127.0), (torch.float8_e4m3fn, 448.0)])
@pytest.mark.parametrize("dtype,residual,shape", [(torch.bfloat16, torch.bfloat16, (3, 7, 2049)), (torch.float32, None, (5, 64)), (torch.float16, torch.float32, (2, 9000)),
                                                  (torch.bfloat16, None, (1, 3))])
def test_norm_in_eight_bits(gpu, quant, limit, dtype, residual, shape):
    """q stands for y to half a step of the 8-bit type: 1/254 of the row's largest value for integers, a 16th of the value (or half the
    smallest step, 2^-10 of the scale) for floats; the scale to fp32's precision."""
    g = torch.Generator().manual_seed(43)
    x, w = torch.randn(shape, generator=g).to(dtype), 1 + 0.2 * torch.randn(shape[-1], generator=g)
    x.view(-1, shape[-1])[0] = 0
    res = None if residual is None else (3 * torch.randn(shape, generator=g)).to(residual)
    if res is not None:
        res.view(-1, shape[-1])[0] = 0
    total = x if res is None else (x.float() + res.float()).to(residual)
    want = total.double() / torch.sqrt(total.double().square().mean(-1, keepdim=True) + 1e-5) * w.double()
    q, scale, *more = f.rms_norm(x.to(gpu), w.to(gpu), None if res is None else res.to(gpu), eps=1e-5, quant=quant)
    assert q.dtype == quant and scale.shape == x.shape[:-1] and len(more) == (res is not None)
    q, scale = q.cpu().double(), scale.cpu().double().unsqueeze(-1)
    most = want.abs().amax(-1, keepdim=True)
    assert torch.all((scale - torch.where(most == 0, 1.0, most / limit)).abs() <= 64 * 2.0 ** -24 * scale)
    step = torch.full_like(want, 0.5) if quant == torch.int8 else torch.maximum(want.abs() / scale / 16, torch.tensor(2.0 ** -10))
    assert torch.all((q * scale - want).abs() <= step * scale * (1 + 1e-4))
    assert (q[want == 0] == 0).all()


def test_norm_rows_that_are_not_finite(gpu):
    x = torch.randn(4, 100)
    x[1, 3], x[2, 5] = float("nan"), float("inf")
    w = torch.ones(100)
    want = x.double() / torch.sqrt(x.double().square().mean(-1, keepdim=True) + 1e-6)
    got = f.rms_norm(x.to(gpu), w.to(gpu)).cpu()
    assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got[2].nan_to_num(7), want[2].float().nan_to_num(7))
    q, scale = f.rms_norm(x.to(gpu), w.to(gpu), quant=torch.float8_e4m3fn)
    assert scale.cpu().isnan().tolist() == [False, True, True, False] and q[0].float().isfinite().all() and q[3].float().isfinite().all()


def test_calls_use_the_current_stream(gpu):
    """Inputs that a stream is still busy with are waited for on that stream, and by a graph's replays."""
    v = make_scan(13, torch.float32, 1, 300, 64, 16)
    d = {k: None if t is None else t.to(gpu) for k, t in v.items()}
    w = torch.randn(64, 4, device=gpu)
    want = f.selective_scan(**dict(d, x=f.causal_conv(f.rms_norm(d["x"], w[:, 0].contiguous()), w)), softplus=True)
    side = torch.cuda.Stream()
    late = torch.empty_like(d["x"])
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        m = torch.randn(2048, 2048, device=gpu)
        for _ in range(20):
            m = m @ m * 1e-3
        late.copy_(d["x"])
        got = f.selective_scan(**dict(d, x=f.causal_conv(f.rms_norm(late, w[:, 0].contiguous()), w)), softplus=True)
    side.synchronize()
    assert torch.equal(got, want)
    graph, x = torch.cuda.CUDAGraph(), torch.zeros_like(d["x"])
    col = w[:, 0].contiguous()
    with torch.cuda.graph(graph):
        out = f.selective_scan(**dict(d, x=f.causal_conv(f.rms_norm(x, col), w)), softplus=True)
    for scale in (1.0, 0.5, 1.0):
        x.copy_(d["x"] * scale)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, f.selective_scan(**dict(d, x=f.causal_conv(f.rms_norm(d["x"] * scale, col), w)), softplus=True))


def test_native_host_path_is_the_python_path(gpu, monkeypatch):
    """Calls take the native host path, and give what the Python one gives; what it does not cover it leaves alone."""
    assert state_space._native is not None
    taken = []

    class Counted:
        def __getattr__(self, name):
            def call(*args):
                out = getattr(state_space.hip._native, name)(*args)
                taken.append((name, out is not None))
                return out
            return call

    def both(fn, *args, covered=True, **kwargs):
        fresh = lambda: ([a.clone() if torch.is_tensor(a) and a.is_contiguous() else a for a in args], kwargs)  # noqa: E731
        outs = []
        for native in (Counted(), None):
            monkeypatch.setattr(state_space, "_native", native)
            a, k = fresh()
            versions = a[0]._version
            out = fn(*a, **k)
            outs.append([*(out if isinstance(out, tuple) else (out,)), *([a[0], torch.tensor(a[0]._version - versions)] if fn.__name__.endswith("step") else [])])
        assert taken.pop()[1] == covered and len(outs[0]) == len(outs[1]), fn.__name__
        for p, q in zip(*outs):
            assert p.dtype == q.dtype and p.shape == q.shape and torch.equal(p.float(), q.float()), fn.__name__

    for dtype in (torch.bfloat16, torch.float32):
        v = make_scan(17, dtype, 0, 0, 40, 16, groups=2, lengths=[70, 0, 33], state=True)
        d = {k: None if t is None else t.to(gpu) for k, t in v.items()}
        args = [d[k] for k in ("x", "dt", "A", "B", "C", "D", "z", "dt_bias")]
        both(f.selective_scan, *args, softplus=True, state=d["state"], offsets=d["offsets"], return_state=True)
        both(f.selective_scan, *args[:5], softplus=True)
        both(f.selective_scan, *args[:3], d["B"][:, :, 0], d["C"][:, :, 0], d["D"], softplus=True)
        both(f.selective_scan, *args[:2], d["A"].t().contiguous().t(), *args[3:], softplus=True, covered=False)
        wide = torch.cat((d["x"], d["z"]), -1)
        both(f.selective_scan, wide[..., :40], d["dt"], *args[2:6], wide[..., 40:], d["dt_bias"], softplus=True)
        token = [None if t is None else t[0, :5] if t.dim() > 2 else t for t in args]
        both(f.selective_scan_step, torch.randn(7, 40, 16, device=gpu), *token, softplus=True, slots=torch.tensor([3, 0, -1, 6, 2], device=gpu))
        both(f.selective_scan_step, torch.randn(5, 40, 16, device=gpu), *token, softplus=True)
        w, b = torch.randn(40, 4, device=gpu), torch.randn(40, device=gpu)
        kept = torch.randn(3, 3, 40, device=gpu).to(dtype)
        both(f.causal_conv, d["x"], w, b, activation="silu", state=kept, offsets=d["offsets"], return_state=True)
        both(f.causal_conv, wide[..., :40], w)
        both(f.causal_conv_step, torch.randn(7, 3, 40, device=gpu).to(dtype), token[0], w, b, activation="silu", slots=torch.tensor([3, 0, -1, 6, 2], dtype=torch.int32, device=gpu))
        for quant in (None, torch.int8, torch.float8_e4m3fn):
            both(f.rms_norm, d["x"], b, quant=quant)
            both(f.rms_norm, wide[..., :40], b, d["z"].float(), quant=quant, eps=1e-3)
        both(f.rms_norm, d["x"].transpose(0, 1).expand(103, 2, 40), b, covered=False)
    with torch.no_grad():
        both(f.rms_norm, d["x"].requires_grad_(), b)
    with pytest.raises(TypeError):
        f.rms_norm(b, b, quant=torch.uint8)


def test_native_autograd_nodes_are_the_python_ones(gpu, monkeypatch):
    """The same gradients, bit for bit, from the nodes in C++ as from those in Python: of every argument or of some, of every output or of
    one, of expanded and transposed gradients; a second derivative is refused by both."""
    native = state_space._native
    assert native is not None

    def both(fn, args, kwargs, some=None, only=None):
        results = []
        for path in (native, None):
            monkeypatch.setattr(state_space, "_native", path)
            leaves = {k: t.detach().clone().requires_grad_(some is None or k in some) if torch.is_tensor(t) and t.is_floating_point() else t for k, t in args.items()}
            out = fn(**leaves, **kwargs)
            out = out if isinstance(out, tuple) else (out,)
            assert all(o.requires_grad for o in out)
            assert ("CppNode" in out[0].grad_fn.name()) == (path is not None), out[0].grad_fn.name()
            torch.manual_seed(5)
            grads = [torch.randn(o.shape, device=gpu).to(o.dtype) for o in out]
            used = range(len(out)) if only is None else [only]
            torch.autograd.backward([out[i] for i in used], [grads[i] for i in used])
            results.append([*out, *(t.grad for t in leaves.values() if torch.is_tensor(t))])
        for p, q in zip(*results):
            assert (p is None) == (q is None) and (p is None or (p.dtype == q.dtype and torch.equal(p, q))), (fn.__name__, some, only)

    for dtype in (torch.bfloat16, torch.float32):
        for offsets in (None, [70, 0, 33]):
            v = make_scan(19, dtype, 2, 103, 40, 16, groups=2, lengths=offsets, state=True)
            d = {k: None if t is None else t.to(gpu) for k, t in v.items()}
            d["A"] = d["A"].to(torch.float32)
            kept = torch.randn(d["state"].shape[0], 3, 40, device=gpu).to(dtype)
            conv = dict(x=d["x"], weight=torch.randn(40, 4, device=gpu).to(dtype), bias=torch.randn(40, device=gpu), state=kept, offsets=d["offsets"])
            for kwargs, only in (({}, None), ({"return_state": True}, None), ({"return_state": True}, 0), ({"return_state": True}, 1)):
                both(f.selective_scan, d, dict(softplus=True, **kwargs), only=only)
                both(f.causal_conv, conv, dict(activation="silu", **kwargs), only=only)
            both(f.selective_scan, {k: None if k in ("z", "D", "dt_bias", "state") else t for k, t in d.items()}, dict(softplus=True), some=("A", "x"))
            both(f.selective_scan, d, dict(softplus=True), some=("state",))
            both(f.causal_conv, dict(conv, bias=None, state=None), {}, some=("weight",))
        x, w, r = torch.randn(3, 5, 40, device=gpu).to(dtype), torch.randn(40, device=gpu), torch.randn(3, 5, 40, device=gpu)
        both(f.rms_norm, dict(x=x, weight=w), {})
        both(f.rms_norm, dict(x=x, weight=w.to(dtype)), {}, some=("weight",))
        for residual in (r, r.to(dtype)):
            for only in (None, 0, 1):
                both(f.rms_norm, dict(x=x, weight=w, residual=residual), dict(eps=1e-3), only=only)
    def spread(t):  # the same values at other strides
        if t.dim() == 0 or t.numel() == 0:
            return t
        out = torch.empty([2 * n for n in t.shape], dtype=t.dtype, device=t.device)[tuple(slice(None, None, 2) for _ in t.shape)]
        return out.copy_(t)

    v = {k: None if t is None else t.to(gpu) for k, t in make_scan(20, torch.float32, 2, 140, 24, 16, groups=2, state=True).items()}
    leaves = [t.requires_grad_() for t in v.values() if t is not None]
    w4, wide = torch.randn(24, 4, device=gpu, requires_grad=True), torch.randn(24, device=gpu, requires_grad=True)
    for path in (native, None):
        monkeypatch.setattr(state_space, "_native", path)
        got = []
        for unpack in (lambda t: t, spread):
            with torch.autograd.graph.saved_tensors_hooks(lambda t: t.detach(), unpack):
                y = f.selective_scan(**dict(v, x=f.causal_conv(f.rms_norm(v["x"], wide), w4, activation="silu")), softplus=True)
            got.append(torch.autograd.grad(y.square().sum(), [*leaves, w4, wide]))
        assert all(torch.equal(p, q) for p, q in zip(*got))
    for path in (native, None):
        monkeypatch.setattr(state_space, "_native", path)
        wide = torch.randn(4, 6, 80, device=gpu, requires_grad=True)
        results = [f.rms_norm(wide[..., :40], w), f.causal_conv(wide[..., 40:], torch.ones(40, 4, device=gpu))]
        total = torch.autograd.grad(sum(t.square().sum() for t in results) + (results[1].transpose(0, 1) * 2).sum(), wide, create_graph=True)[0]
        with pytest.raises(RuntimeError, match="differentiate twice|once_differentiable"):
            total.square().sum().backward()


def test_calls_on_a_device_that_is_not_current_and_errors(gpu):
    with pytest.raises(RuntimeError, match="on cpu"):
        f.rms_norm(torch.ones(3, device=gpu), torch.ones(3))
    with pytest.raises(RuntimeError, match="on cpu"):
        f.causal_conv_step(torch.ones(1, 3, 2), torch.ones(1, 2, device=gpu), torch.ones(2, 4, device=gpu))
