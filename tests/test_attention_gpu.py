"""
The linear attention layer's kernels against the plain loops of scanscam_amd.baseline in float64 on the same stored inputs, gradients
against those that torch.autograd takes of these loops.

Bounds. Every output is a sum of products, of which the same call on the inputs' absolute values (and its gradients) gives the sum of absolute values, A.
With h half a unit in the last place of the activations' type, relative (2^-8 bf16, 2^-11 fp16, 2^-24 fp32):
  * each product passes up to two roundings to that type on its way (its score's; or where no state is handed over that of what is added to the state,
    and the state's): 2 h A; and the result one more: h |want|;
  * in fp32 a product is rounded once for each addition on its way, at most K + V + C + 2 T of them and some 64 of exponentials and factors:
    (600 + 2 T) 2^-24 A;
  * float32 results (states, gradients of states and of decays) have no rounding to the type, but two terms of it, 2^-17 A (bf16; fp16 2^-21);
  * a decay's gradient is what passes its token, out of running sums (in fp64) from the sequence's end on of what later tokens read less what they
    write. These terms' own errors stay in the sums where the terms themselves cancel, as at a first token, whose gradient is zero: a chunk of 32
    tokens or more adds its terms' (K + V + C + 64) 2^-24 of what crosses its borders, independent ones, so that the largest A of the head takes A's place.
fp16's smallest steps add 2^-16 of the largest A: a score below 2^-14 is rounded in steps of 2^-24, times up to 64 values.
"""
import pytest
import torch

import scanscam_amd as f
from scanscam_amd import attention, baseline

pytestmark = pytest.mark.gpu

HALF = {t: torch.finfo(t).eps / 2 for t in (torch.float32, torch.bfloat16, torch.float16)}
TERMS = {torch.float32: 0.0, torch.bfloat16: 2.0 ** -17, torch.float16: 2.0 ** -21}


def close(got, want, total, dtype, T, what, exact=False):
    """``total``: A; ``dtype``: of the activations; ``exact``: a float32 result, whatever type it is handed over in."""
    assert got.shape == want.shape, (what, got.shape, want.shape)
    if got.numel() == 0:
        return
    half = HALF[got.dtype]
    got, want, total = got.detach().cpu().double(), want.detach().cpu().double(), total.detach().cpu().double()
    assert torch.isfinite(got).all(), what
    bound = 1.01 * half * want.abs() + (600 + 2 * T) * 2.0 ** -24 * total + (TERMS[dtype] if exact else 2.02 * HALF[dtype]) * total
    if dtype == torch.float16:
        bound = bound + 2.0 ** -16 * total.max()
    over = (got - want).abs() - bound
    at = int(over.argmax())
    if (over > 0).any():
        pytest.fail(f"{what}: {float((got - want).abs().max()):.3e} off; at {at}: {float(got.flatten()[at])} for {float(want.flatten()[at])}, bound {float(bound.expand_as(over).flatten()[at]):.3e}")


def offsets_of(lengths, dtype=torch.int32):
    return torch.tensor([0] + torch.tensor(lengths).cumsum(0).tolist(), dtype=dtype)


def make(seed, dtype, batch, T, heads, K, V, groups=None, decay="token", lengths=None, state=False, logs=torch.float32, pace=0.1):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(s, generator=g)  # noqa: E731
    if lengths is not None:
        batch, T = 1, sum(lengths)
    groups = groups or heads
    v = {"q": r(batch, T, groups, K).to(dtype), "k": r(batch, T, groups, K).to(dtype), "v": r(batch, T, heads, V).to(dtype)}
    rate = torch.exp(r(heads)) * pace
    v["decay"] = None if decay is None else (-rate).to(logs) if decay == "head" else (-rate * r(batch, T, heads).abs()).to(logs)
    v["state"] = r(batch if lengths is None else len(lengths), heads, K, V) if state else None
    v["offsets"] = offsets_of(lengths) if lengths is not None else None
    return v


def wide(t):
    return t if t is None or not t.is_floating_point() else t.double()


def sizes(t, name):
    """Absolute values, but of decays, which are exponents."""
    return t if t is None or name in ("decay", "offsets") else t.abs()


CASES = [
    # dtype, batch, T, heads, K, V, and what differs
    (torch.float32, 2, 100, 3, 16, 16, {}),
    (torch.float32, 1, 1, 1, 1, 1, {"state": True}),
    (torch.float32, 2, 0, 2, 8, 4, {"state": True}),
    (torch.float32, 1, 33, 2, 48, 72, {"decay": "head", "state": True}),
    (torch.float32, 1, 70, 4, 128, 100, {"groups": 2}),
    (torch.float32, 1, 65, 2, 130, 256, {"state": True}),
    (torch.float32, 0, 0, 2, 24, 20, {"lengths": [1, 0, 64, 0, 33, 130, 0], "state": True}),
    (torch.float32, 2, 40, 2, 31, 7, {"decay": None}),
    (torch.bfloat16, 2, 130, 2, 64, 64, {"state": True}),
    (torch.bfloat16, 1, 200, 4, 128, 128, {"groups": 1, "state": True}),
    (torch.bfloat16, 2, 129, 2, 127, 65, {}),
    (torch.bfloat16, 1, 70, 1, 256, 200, {"state": True}),
    (torch.bfloat16, 0, 0, 3, 32, 128, {"lengths": [64, 5, 0, 300, 1], "state": True}),
    (torch.bfloat16, 1, 64, 2, 16, 8, {"logs": torch.bfloat16, "decay": "head"}),
    (torch.bfloat16, 1, 300, 2, 128, 64, {"pace": 30.0, "state": True}),
    (torch.float16, 2, 150, 2, 64, 128, {"groups": 1, "state": True}),
    (torch.float16, 1, 90, 2, 80, 33, {"logs": torch.float16}),
    (torch.float16, 0, 0, 1, 256, 256, {"lengths": [0, 100, 28], "state": True}),
    (torch.bfloat16, 1, 777, 2, 64, 64, {"pace": 0.001, "state": True}),
    (torch.float32, 2, 700, 2, 16, 24, {"state": True}),
    (torch.float16, 0, 0, 2, 32, 16, {"lengths": [600, 3, 1200, 513], "state": True}),
]


@pytest.mark.parametrize("dtype,batch,T,heads,K,V,more", CASES, ids=lambda v: str(v).replace("torch.", "").replace(" ", ""))
@pytest.mark.parametrize("parts,native", [(0, True), (0, False), (1, False), (3, False)])
def test_attention_and_gradients(gpu, monkeypatch, dtype, batch, T, heads, K, V, more, parts, native):
    monkeypatch.setattr(attention, "_parts", parts)  # parts of time to share out, also where there is less than a chunk for each
    if not native:  # the host path in Python
        monkeypatch.setattr(attention, "_native", None)
    v, scale = make(5, dtype, batch, T, heads, K, V, **more), K ** -0.5
    state = v["state"] is not None
    names = [n for n, t in v.items() if t is not None and n != "offsets"]
    g = torch.Generator().manual_seed(6)
    gy, gs = torch.randn(v["v"].shape, generator=g).to(dtype), torch.randn((v["state"] if state else torch.zeros(0)).shape, generator=g)

    def reference(of, gy, gs):
        ref = {n: of(wide(t), n).requires_grad_() if n in names else t for n, t in v.items()}
        y, new = baseline.naive_linear_attention(**ref, scale=scale, return_state=True)
        outs, weights = ((y, new), (gy, gs)) if state else ((y,), (gy,))
        grads = torch.autograd.grad(outs, [ref[n] for n in names], weights, allow_unused=True)
        return y, new, [torch.zeros(v[n].shape, dtype=torch.float64) if d is None else d for n, d in zip(names, grads)]

    want, want_state, want_grads = reference(lambda t, n: t, gy.double(), gs.double())
    size, size_state, size_grads = reference(sizes, gy.double().abs(), gs.double().abs())
    dev = {n: None if t is None else t.to(gpu).requires_grad_(n in names) for n, t in v.items()}
    with torch.no_grad():
        plain = f.linear_attention(**dev, scale=scale)
    got = f.linear_attention(**dev, scale=scale, return_state=state)
    got, got_state = got if state else (got, None)
    Tn = v["v"].shape[1]
    assert state or torch.equal(plain, got.detach())
    close(plain, want, size, dtype, Tn, "y of a call without gradients")
    close(got, want, size, dtype, Tn, "y")
    if state:
        close(got_state, want_state, size_state, dtype, Tn, "state", exact=True)
    outs, weights = ((got, got_state), (gy.to(gpu), gs.to(gpu))) if state else ((got,), (gy.to(gpu),))
    grads = torch.autograd.grad(outs, [dev[n] for n in names], weights, retain_graph=True)
    again = torch.autograd.grad(outs, [dev[n] for n in names], weights)
    for n, a, b, w, s in zip(names, grads, again, want_grads, size_grads):
        assert a.dtype == v[n].dtype and torch.equal(a, b), n  # (the order of every sum is fixed)
        if n == "decay" and s.dim() == 3 and s.numel():
            s = s.amax(1, keepdim=True).expand_as(s)
        close(a, w, s, dtype, Tn, f"gradient of {n}", exact=n in ("decay", "state"))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows,heads,K,V,groups,decay", [(1, 1, 1, 1, 1, "token"), (3, 2, 16, 16, 1, "token"), (5, 3, 33, 65, 3, "head"), (2, 4, 128, 128, 2, None),
                                                         (2, 1, 256, 256, 1, "token"), (70, 2, 8, 130, 2, "token"), (1, 16, 128, 128, 16, "token")])
@pytest.mark.parametrize("wide_slots,native", [(True, True), (False, True), (False, False)])
def test_attention_step(gpu, monkeypatch, dtype, rows, heads, K, V, groups, decay, wide_slots, native):
    if not native:
        monkeypatch.setattr(attention, "_native", None)
    v = make(8, dtype, rows, 1, heads, K, V, groups, decay)
    slots = torch.randperm(rows + 4, generator=torch.Generator().manual_seed(1))[:rows]
    if rows > 2:
        slots[1], slots[2] = -1, rows + 4  # rows without a sequence
    slots = slots.to(torch.int64 if wide_slots else torch.int32)
    state = torch.randn(rows + 4, heads, K, V, generator=torch.Generator().manual_seed(2))
    args = [v[n] if v[n] is None or v[n].dim() == 1 else v[n][:, 0] for n in ("q", "k", "v", "decay")]
    results = []
    for of in (lambda t, n: t, sizes):
        new = of(state.double(), "state")
        y = baseline.naive_linear_attention_step(new, *[of(wide(t), n) for t, n in zip(args, ("q", "k", "v", "decay"))], scale=0.7, slots=slots)
        results.append((y, new))
    dev = state.to(gpu)
    got = f.linear_attention_step(dev, *[None if t is None else t.to(gpu) for t in args], scale=0.7, slots=slots.to(gpu))
    for a, b, c, what in zip((got, dev), *results, ("y", "state")):
        close(a, b, c, torch.float32, 1, what)
    untouched = [s for s in range(rows + 4) if s not in slots.tolist()]
    assert torch.equal(dev[untouched].cpu(), state[untouched])


# dtype, rows, channels, groups, weight and bias, gate, activation
NORMS = [
    (torch.float32, 5, 12, 3, True, True, None),
    (torch.float32, 1, 1, 1, True, False, "silu"),
    (torch.float32, 700, 96, 4, True, False, None),
    (torch.float32, 3, 2000, 1, True, True, "silu"),
    (torch.float32, 9, 8192, 1, False, True, None),
    (torch.bfloat16, 300, 2048, 16, True, True, None),
    (torch.bfloat16, 70, 2050, 10, True, True, "silu"),
    (torch.bfloat16, 11, 7, 7, True, False, None),
    (torch.bfloat16, 5, 4100, 2, False, False, None),
    (torch.bfloat16, 4, 8191, 1, True, True, None),
    (torch.float16, 33, 1536, 3, True, True, None),
    (torch.float16, 20, 40, 20, False, False, "silu"),
    (torch.float16, 1300, 24, 1, True, True, None),
]


def norm_close(got, want, what, terms=1.0):
    """h |want| of the result's own rounding; in fp32 some 64 roundings at the size of the largest value of the result, ``terms`` for sums over rows."""
    assert got.shape == want.shape, what
    half = HALF[got.dtype]
    got, want = got.detach().cpu().double(), want.detach().double()
    bound = 1.01 * half * want.abs() + 64 * 2.0 ** -24 * terms * want.abs().max()
    if half == HALF[torch.float16]:
        bound = bound + 2.0 ** -25
    assert torch.isfinite(got).all() and ((got - want).abs() <= bound).all(), f"{what}: {float(((got - want).abs() - bound).max()):.3e} over, of {float(want.abs().max()):.3e}"


@pytest.mark.parametrize("dtype,rows,channels,groups,affine,gate,activation", NORMS, ids=lambda v: str(v).replace("torch.", ""))
@pytest.mark.parametrize("native", [True, False])
def test_group_norm_and_gradients(gpu, monkeypatch, dtype, rows, channels, groups, affine, gate, activation, native):
    if not native:
        monkeypatch.setattr(attention, "_native", None)
    g = torch.Generator().manual_seed(3)
    r = lambda *s: torch.randn(s, generator=g)  # noqa: E731
    v = {"x": (r(rows, channels) * 3 + 1).to(dtype), "weight": r(channels) + 1 if affine else None, "bias": r(channels) if affine else None,
         "z": r(rows, channels).to(dtype) if gate else None}
    names, gy = [n for n, t in v.items() if t is not None], r(rows, channels).to(dtype)
    ref = {n: None if t is None else t.double().requires_grad_() for n, t in v.items()}
    want = baseline.naive_group_norm(ref["x"], groups, ref["weight"], ref["bias"], ref["z"], activation=activation)
    want_grads = torch.autograd.grad(want, [ref[n] for n in names], gy.double())
    dev = {n: None if t is None else t.to(gpu).requires_grad_() for n, t in v.items()}
    call = lambda: f.group_norm(dev["x"], groups, dev["weight"], dev["bias"], dev["z"], activation=activation)  # noqa: E731
    with torch.no_grad():
        plain = call()
    got = call()
    assert torch.equal(plain, got.detach())
    norm_close(got, want, "y")
    grads, again = (torch.autograd.grad(call(), [dev[n] for n in names], gy.to(gpu)) for _ in range(2))
    for n, a, b, w in zip(names, grads, again, want_grads):
        assert a.dtype == v[n].dtype and torch.equal(a, b), n
        if channels // groups > 1 or n != "x":  # (a channel alone is its own mean: its gradient is zero)
            norm_close(a, w, f"gradient of {n}", terms=rows ** 0.5 if n in ("weight", "bias") else 1.0)
        else:
            assert a.float().abs().max() <= 2.0 ** -16 * 316.3 * float(gy.float().abs().max()) * 16


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_float32_results_of_16_bits_are_float32_s(gpu, dtype):
    """
    States and gradients of decays, over all values together: no term of a product is lost. What a token reads or writes is a sum whose products pass some 40
    roundings of 2^-24, independent ones: 40^0.5 2^-24 = 3.8e-7 of it. A decay's gradient is a running sum of such terms over 8 chunks, of two kinds each, which
    cancel to about the size of one: 16^0.5 as much, 1.5e-6, below 2^-19. (A product's second term that is missing costs 2^-11 of one product in some 10^4.)
    """
    v = make(12, dtype, 2, 512, 4, 128, 64, groups=2, state=True)
    names = [n for n, t in v.items() if t is not None]
    ref, dev = {n: wide(v[n]).requires_grad_() for n in names}, {n: v[n].to(gpu).requires_grad_() for n in names}
    outs, grads = [], []
    for call, leaves in ((baseline.naive_linear_attention, ref), (f.linear_attention, dev)):
        y, state = call(**leaves, scale=0.1, return_state=True)
        outs.append(state)
        weights = [torch.linspace(-1, 1, t.numel(), dtype=torch.float64).view(t.shape) for t in (y, state)]
        grads.append(torch.autograd.grad((y, state), [leaves["decay"], leaves["state"]], [w.to(dtype).to(t) if t is y else w.float().to(t) for w, t in zip(weights, (y, state))]))
    for want, got in [outs] + list(zip(*grads)):
        assert (got.detach().cpu().double() - want.detach()).norm() <= 2.0 ** -19 * want.detach().norm()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("parts", [0, 7, 45, 200])
def test_long_and_short_sequences_behind_each_other(gpu, monkeypatch, dtype, parts):
    """A long one is shared out in more parts than a short one."""
    test_attention_and_gradients(gpu, monkeypatch, dtype, 0, 0, 2, 32, 24, {"lengths": [1, 0, 900, 64, 3, 2000, 130, 0], "state": True}, parts, False)


def test_more_sequences_than_a_wave_counts_at_once(gpu, monkeypatch):
    lengths = [(7 * i) % 40 for i in range(150)]
    lengths[70], lengths[149] = 700, 300
    test_attention_and_gradients(gpu, monkeypatch, torch.bfloat16, 0, 0, 2, 16, 20, {"lengths": lengths, "state": True}, 0, True)
    test_attention_and_gradients(gpu, monkeypatch, torch.bfloat16, 0, 0, 2, 16, 20, {"lengths": lengths, "state": True}, 20, False)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("K,V", [(200, 27), (61, 199), (101, 30), (5, 90), (130, 3)])
@pytest.mark.parametrize("T,parts", [(70, 0), (203, 2)])
def test_one_side_half_as_wide_or_less(gpu, monkeypatch, dtype, K, V, T, parts):
    """Waves hold half as many columns where a side leaves half of them empty."""
    test_attention_and_gradients(gpu, monkeypatch, dtype, 2, T, 2, K, V, {"groups": 1, "state": True}, parts, False)
