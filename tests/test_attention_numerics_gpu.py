"""
The attention's kernels where numbers are small, large, or of very different sizes: against the plain loops in float64 on the same stored inputs.

Bounds. With A the sum of an output's products' absolute values (as in test_attention_gpu.py) and h half a unit in the last place of the activations' type, relative:
  * a float32 factor of a product is taken apart into terms of the type, two at least: 2^-17 (bf16) or 2^-22 (fp16) of it is lost, at up to two places of a chain
    of products (what is added to a state, and the state or the score that is read): TERMS A;
  * in fp32 a product is rounded once for each addition on its way, at most K + V + C + 2 T of them and some 64 of exponentials and factors: (600 + 2 T) 2^-24 A;
  * a result in 16 bits is rounded once: h |want|, in fp16 2^-25 at least (half of its smallest step).
"""
import math

import pytest
import torch

import scanscam_amd as f
from scanscam_amd import attention, baseline
from test_attention_gpu import HALF, make, sizes, wide

pytestmark = pytest.mark.gpu

TERMS = {torch.float32: 0.0, torch.bfloat16: 2.0 ** -16, torch.float16: 2.0 ** -21}
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def call(attend, given, names, scale, gy=None, gs=None):
    """(y, new state, gradients by name); ``gs`` None: no gradient of the new state."""
    y, new = attend(**given, scale=scale, return_state=True)
    if gy is None:
        return y.detach(), new.detach(), {}
    outs, weights = ([y], [gy]) if gs is None else ([y, new], [gy, gs])
    grads = torch.autograd.grad(outs, [given[n] for n in names], weights, allow_unused=True)
    return y.detach(), new.detach(), {n: torch.zeros_like(given[n]) if t is None else t for n, t in zip(names, grads)}


def results(gpu, given, scale, gy=None, gs=None):
    """The kernels' results, what is right, and A of each."""
    names = [n for n, t in given.items() if t is not None and n != "offsets"]
    out = []
    for attend, of, weight in ((f.linear_attention, lambda t, n: t.to(gpu), lambda t: t.to(gpu)), (baseline.naive_linear_attention, lambda t, n: wide(t), wide),
                               (baseline.naive_linear_attention, lambda t, n: sizes(wide(t), n), lambda t: wide(t).abs())):
        own = {n: None if t is None else of(t, n).requires_grad_() if n in names and gy is not None else of(t, n) for n, t in given.items()}
        out.append(call(attend, own, names, scale, None if gy is None else weight(gy), None if gs is None else weight(gs)))
    return out


def near(got, want, total, dtype, T, what):
    """``total``: A."""
    assert got.shape == want.shape and torch.isfinite(got).all(), what
    half = HALF[got.dtype]
    got, want, total = got.detach().cpu().double(), want.detach().cpu().double(), total.detach().cpu().double()
    bound = 1.01 * half * want.abs() + ((600 + 2 * T) * 2.0 ** -24 + TERMS[dtype]) * total + (2.0 ** -25 if half == HALF[torch.float16] else 0.0)
    over = (got - want).abs() - bound
    at = int(over.argmax())
    assert not (over > 0).any(), f"{what}: {float((got - want).abs().max()):.3e} off; at {at}: {float(got.flatten()[at])} for {float(want.flatten()[at])}, bound {float(bound.flatten()[at]):.3e}"


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("K,V,T,groups", [(64, 64, 300, 2), (128, 128, 200, 1), (128, 64, 130, 2), (256, 200, 100, 1), (33, 97, 140, 2)])
@pytest.mark.parametrize("parts", [0, 2])
def test_results_in_16_bits_are_rounded_once(gpu, monkeypatch, dtype, K, V, T, groups, parts):
    """Whatever is asked for besides: outputs have the same bits with a state handed back, with gradients, and without either."""
    monkeypatch.setattr(attention, "_parts", parts)
    v, scale = make(23, dtype, 2, T, 2, K, V, groups=groups, pace=0.02, state=True), K ** -0.5
    gy = torch.randn(v["v"].shape, generator=torch.Generator().manual_seed(24)).to(dtype)
    got, want, total = results(gpu, v, scale, gy)
    near(got[0], want[0], total[0], dtype, T, "y")
    for n in ("q", "k", "v"):
        near(got[2][n], want[2][n], total[2][n], dtype, T, f"gradient of {n}")
    alone = f.linear_attention(**{n: t if t is None else t.to(gpu) for n, t in v.items()}, scale=scale)
    assert torch.equal(alone, got[0])



@pytest.mark.parametrize("qk,vs,gs", [(1e-3, 100.0, 1.0), (3e-4, 1000.0, 0.1), (1e-4, 6000.0, 0.01), (1.0, 1.0, 1e-5), (1.0, 1.0, 1e-6), (40.0, 10.0, 1e-3)])
@pytest.mark.parametrize("K,V,T,parts", [(128, 128, 64, 0), (64, 48, 150, 2), (200, 256, 70, 0)])
def test_products_of_small_and_large_values_in_fp16(gpu, monkeypatch, qk, vs, gs, K, V, T, parts):
    """Products of queries and keys, or of gradients and values, far below fp16's smallest steps, or past its largest value, where results are neither."""
    monkeypatch.setattr(attention, "_parts", parts)
    v, scale = make(21, torch.float16, 1, T, 2, K, V, groups=1, pace=0.02), 1.0 if qk < 1 else K ** -0.5
    v["q"], v["k"], v["v"] = (v["q"].float() * qk).half(), (v["k"].float() * qk).half(), (v["v"].float() * vs).half()
    if qk > 1:
        scale = 1e-3  # (products of 40 x 40 x 128 are more than fp16 holds; what comes of them is not)
        v["q"] *= 4
    gy = (torch.randn(v["v"].shape, generator=torch.Generator().manual_seed(22)) * gs).half()
    got, want, total = results(gpu, v, scale, gy)
    near(got[0], want[0], total[0], torch.float16, T, "y")
    near(got[1], want[1], total[1], torch.float16, T, "state")
    for n in ("q", "k", "v"):
        near(got[2][n], want[2][n], total[2][n], torch.float16, T, f"gradient of {n}")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("parts", [0, 2])
@pytest.mark.parametrize("size", [1.0, 2.0 ** -6])
def test_states_grow_as_far_as_float32_holds_them(gpu, monkeypatch, dtype, parts, size):
    """Decays above zero: states of some 1e36, and gradients of states as large, to which tokens before and after add as little as ever."""
    monkeypatch.setattr(attention, "_parts", parts)
    T = 200
    v = make(25, dtype, 1, T, 2, 48, 64, state=True)
    v["v"], v["q"] = (v["v"].float() * size).to(dtype), (v["q"].float() * size).to(dtype)
    v["decay"] = torch.zeros(1, T, 2)
    v["decay"][:, 65:135] = 83.0 / 70
    g = torch.Generator().manual_seed(26)
    gy, gs = torch.randn(v["v"].shape, generator=g).to(dtype), torch.randn(v["state"].shape, generator=g)
    found = []
    for attend, of, weight in ((f.linear_attention, lambda t, n: t.to(gpu), lambda t: t.to(gpu)), (baseline.naive_linear_attention, lambda t, n: wide(t), wide),
                               (baseline.naive_linear_attention, lambda t, n: sizes(wide(t), n), lambda t: wide(t).abs())):
        given = {n: t if t is None else of(t, n).requires_grad_(n == "state") for n, t in v.items()}
        y, new = attend(**given, return_state=True)  # (what queries read of it is more than fp16 holds)
        found.append((new.detach(), *torch.autograd.grad((y, new), given["state"], (weight(gy), weight(gs)))))
    for got, want, total, what in zip(*found, ("state", "gradient of the state")):
        assert want.abs().max() > 1e36
        near(got, want, total, dtype, T, what)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("parts", [0, 2, 3])
def test_decays_of_a_part_grow_past_float32_where_states_do_not(gpu, monkeypatch, dtype, parts):
    """Over hundreds of tokens decays may grow by more than float32 holds: a state of zero, and a gradient of zero, stay what they are."""
    monkeypatch.setattr(attention, "_parts", parts)
    T = 900
    v = make(27, dtype, 1, T, 2, 40, 24)
    v["decay"] *= 0.01
    v["decay"][:, :256] = 0.5  # e^128 in 256 tokens that add nothing
    v["k"][:, :256] = 0
    got, want, total = results(gpu, v, 0.2)
    near(got[0], want[0], total[0], dtype, T, "y")
    near(got[1], want[1], total[1], dtype, T, "state")
    v = make(28, dtype, 1, T, 2, 40, 24)
    v["decay"] *= 0.01
    v["decay"][:, 640:] = 0.5  # and in as many that are not read, of a state that is zero
    v["decay"][:, 639] = -math.inf
    v["k"][:, 639:] = v["q"][:, 639:] = 0
    gy = torch.randn(v["v"].shape, generator=torch.Generator().manual_seed(29)).to(dtype)
    got, want, total = results(gpu, v, 0.2, gy)
    for n in ("q", "k", "v"):
        near(got[2][n], want[2][n], total[2][n], dtype, T, f"gradient of {n}")


def passing(total, decay, dtype, begin=0, end=None):
    """
    A decay's gradient is the product of state and gradient that passes its chunk, and what passes the token and not the whole chunk. The former comes from the
    product at the next border, eight chunks on at most, less what the tokens between it write and more what they read: what these sums' roundings leave is relative to the largest product on the way, but no
    more than what state and gradient can have as a product: nothing where the chunk's decays let nothing through. That largest product by token, in units of A.
    """
    chunk = 32 if dtype == torch.float32 else 64
    end = total.shape[1] if end is None else end
    out = torch.zeros_like(total)
    chunks = (end - begin + chunk - 1) // chunk
    most = torch.zeros_like(total[:, 0])
    for c in range(chunks - 1, -1, -1):
        a, b = begin + c * chunk, min(begin + (c + 1) * chunk, end)
        if (c + 1) % 8 == 0:  # a border behind this chunk
            most = total[:, b:min(b + 1, end)].amax(1) if b < end else torch.zeros_like(most)
        here = torch.maximum(most, total[:, a:b].amax(1))
        closed = torch.isinf(decay[:, a:b]).any(1)
        out[:, a:b] = torch.where(closed, 0.0, here)[:, None]
        most = torch.where(closed, total[:, a], here)
    return out


def near_decays(got, want, total, decay, dtype, T, what, spans=None):
    """``spans``: first tokens and ends of packed sequences."""
    got, want, total = (t.detach().cpu().double() for t in (got, want, total))
    assert torch.isfinite(got).all()
    noise = torch.zeros_like(total)
    for a, b in spans or [(0, total.shape[1])]:
        noise[:, a:b] = passing(total, decay, dtype, a, b)[:, a:b]
    bound = ((600 + 2 * T) * 2.0 ** -24 + TERMS[dtype]) * (total + noise) + 2.0 ** -44 * total.max() + 1.01 * HALF[torch.float32] * want.abs()
    over = (got - want).abs() - bound
    at = int(over.argmax())
    assert not (over > 0).any(), f"{what}: at {at} of {tuple(got.shape)}: {float(got.flatten()[at])} for {float(want.flatten()[at])}, bound {float(bound.flatten()[at]):.3e}"


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("T,cut", [(64, 20), (40, 39), (700, 300), (1200, 511), (1200, 512)])
@pytest.mark.parametrize("strong", [-math.inf, -90.0])
@pytest.mark.parametrize("K,V", [(64, 64), (24, 128)])
def test_a_decay_s_gradient_is_of_what_passes_it(gpu, dtype, T, cut, strong, K, V):
    """Where a decay lets nothing through its gradient is nothing, however large what later tokens read and write."""
    v = make(31, dtype, 1, T, 2, K, V, pace=0.01)
    v["decay"][0, cut] = strong
    later = min(cut + 12, T - 1)
    v["v"][:, later:] = (v["v"][:, later:].float() * 100).to(dtype)
    gy = torch.randn(v["v"].shape, generator=torch.Generator().manual_seed(32)).to(dtype)
    got, want, total = results(gpu, v, K ** -0.5, gy)
    shown = torch.where(v["decay"] < -80, -math.inf, v["decay"])  # (e^-90 is 2^-130: of products below 2^60, nothing that the bound's last term does not hold)
    near_decays(got[2]["decay"], want[2]["decay"], total[2]["decay"], shown, dtype, T, "gradient of the decays")


# (more than eight chunks: decays' gradients take the product of state and gradient anew at each eighth border, with states that another pass stored)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("K,V,lengths", [(128, 128, None), (128, 64, [1100, 0, 37, 600]), (64, 128, None), (256, 256, None), (130, 40, [3, 1070]), (40, 250, None)])
def test_gradients_of_decays_past_borders_of_wide_heads(gpu, monkeypatch, dtype, K, V, lengths):
    T = sum(lengths) if lengths else 1100
    heads = 1 if K * V > 128 * 128 else 2
    v = make(33, dtype, 1, T, heads, K, V, groups=1, lengths=lengths, state=True, pace=0.002)
    gy = torch.randn(v["v"].shape, generator=torch.Generator().manual_seed(34)).to(dtype)
    gs = torch.randn(v["state"].shape, generator=torch.Generator().manual_seed(35))
    got, want, total = results(gpu, v, K ** -0.5, gy, gs)
    ends = [0] + torch.tensor(lengths).cumsum(0).tolist() if lengths else [0, T]
    spans = list(zip(ends, ends[1:]))
    for parts in (0, 1, 3):
        monkeypatch.setattr(attention, "_parts", parts)
        names = [n for n, t in v.items() if t is not None and n != "offsets"]
        dev = {n: None if t is None else t.to(gpu).requires_grad_(n != "offsets") for n, t in v.items()}
        y, new, grads = call(f.linear_attention, dev, names, K ** -0.5, gy.to(gpu), gs.to(gpu))
        near(y, want[0], total[0], dtype, T, f"y, {parts} parts")
        near(new, want[1], total[1], dtype, T, f"state, {parts} parts")
        for n in ("q", "k", "v", "state"):
            near(grads[n], want[2][n], total[2][n], dtype, T, f"gradient of {n}, {parts} parts")
        near_decays(grads["decay"], want[2]["decay"], total[2]["decay"], v["decay"], dtype, T, f"gradient of decays, {parts} parts", spans)


@pytest.mark.parametrize("dtype,T,K,V,decay", [(torch.bfloat16, 1500, 128, 64, "head"), (torch.float32, 1100, 64, 128, "head"), (torch.float32, 17000, 4, 4, "token"), (torch.float32, 17000, 4, 4, "head")])
def test_gradients_of_decays_over_many_tokens(gpu, dtype, T, K, V, decay):
    """Decays of heads are sums over more than 1024 tokens; and more than 64 times eight chunks of one sequence."""
    v = make(36, dtype, 1, T, 2, K, V, decay="token", pace=0.002)
    if decay == "head":
        v["decay"] = v["decay"][0, 0].clone()
    gy = torch.randn(v["v"].shape, generator=torch.Generator().manual_seed(37)).to(dtype)
    got, want, total = results(gpu, v, K ** -0.5, gy)
    for n in ("q", "k", "v"):
        near(got[2][n], want[2][n], total[2][n], dtype, T, f"gradient of {n}")
    if decay == "head":  # (sums over the tokens in float32 at up to 64 in a row: the products' own roundings are more)
        near(got[2]["decay"], want[2]["decay"], total[2]["decay"], dtype, T, "gradient of the decays")
    else:
        near_decays(got[2]["decay"], want[2]["decay"], total[2]["decay"], v["decay"], dtype, T, "gradient of the decays")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("parts", [0, 3])
def test_states_near_float32_s_largest_value(gpu, monkeypatch, dtype, parts):
    """They decay a little, in one part or from part to part, and stay finite on the way."""
    monkeypatch.setattr(attention, "_parts", parts)
    T = 200
    v = make(38, dtype, 1, T, 2, 24, 16, state=True)
    v["q"] *= 0
    v["state"] = v["state"].sign() * 3.2e38
    v["decay"] = torch.full((1, T, 2), -1e-3)
    gs = v["state"].flip(-1).contiguous()
    given = {n: t if t is None else t.to(gpu).requires_grad_(n == "state") for n, t in v.items()}
    _, new = f.linear_attention(**given, return_state=True)
    back, = torch.autograd.grad(new, given["state"], gs.to(gpu))
    want = v["state"].double() * math.exp(-1e-3 * T)
    near(new, want, want.abs(), dtype, T, "state")
    near(back, want.flip(-1), want.abs(), dtype, T, "gradient of the state")


@pytest.mark.parametrize("K,V,T,parts", [(3, 3, 17, 0), (64, 32, 142, 2), (130, 200, 60, 0)])
def test_small_additions_to_states_in_fp16(gpu, monkeypatch, K, V, T, parts):
    """Gradients of states that nothing but the far ends of a strong decay adds to, and small states: as small as they are."""
    monkeypatch.setattr(attention, "_parts", parts)
    v = make(39, torch.float16, 1, T, 2, K, V, state=True, pace=0.01)
    v["state"] *= 1e-12
    v["decay"][:, 0] = -25.0  # (what reaches the first state is e^-25)
    v["v"] = (v["v"].float() * 1e-3).half()
    g = torch.Generator().manual_seed(40)
    gy, gs = torch.randn(v["v"].shape, generator=g).half(), torch.randn(v["state"].shape, generator=g) * 1e-12
    got, want, total = results(gpu, v, K ** -0.5, gy, gs)
    near(got[1], want[1], total[1], torch.float16, T, "state")
    near(got[2]["state"], want[2]["state"], total[2]["state"], torch.float16, T, "gradient of the state")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("lengths", [[1, 1, 0, 1], [1, 90, 5, 300, 64], [700, 3]])
@pytest.mark.parametrize("parts", [0, 2])
def test_a_first_token_s_decay_has_no_gradient_without_a_state(gpu, monkeypatch, dtype, lengths, parts):
    """There is nothing that it lets through, whatever the last states' gradients are."""
    monkeypatch.setattr(attention, "_parts", parts)
    v = make(41, dtype, 0, 0, 2, 40, 56, lengths=lengths, pace=0.01)
    given = {n: t if t is None else t.to(gpu).requires_grad_(n != "offsets") for n, t in v.items()}
    y, new = f.linear_attention(**given, return_state=True)
    g = torch.Generator().manual_seed(42)
    gy, gs = torch.randn(y.shape, generator=g).to(dtype).to(gpu), torch.randn(new.shape, generator=g).to(gpu)
    grad, = torch.autograd.grad((y, new), given["decay"], (gy, gs))
    first = [int(o) for o, n in zip(v["offsets"], lengths) if n > 0]
    assert grad[0, first].abs().max() <= 2.0 ** -44 * 40 * 56 * 300  # (sums in 64 bits of pairs, of as many products of some 1 each)
    assert all(n < 2 or grad[0, int(o) + 1:int(o) + n].abs().max() > 1e-3 for o, n in zip(v["offsets"], lengths))
