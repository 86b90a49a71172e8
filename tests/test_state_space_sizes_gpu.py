"""
The state space layer's operators at sizes that few calls have: none of something, very many of something, tensors far apart.
"""
import pytest
import torch

import scanscam_amd as f
from scanscam_amd import baseline, state_space

pytestmark = pytest.mark.gpu


def spoil(gpu, numbers):
    """Leaves memory that the next allocations get in a state that is not zeros."""
    for n in numbers:
        torch.full((n,), float("nan"), device=gpu)


def test_selections_of_no_channels_have_gradients_of_zero(gpu):
    B, C = (torch.randn(2, 5, 4, device=gpu, requires_grad=True) for _ in range(2))
    y = f.selective_scan(torch.empty(2, 5, 0, device=gpu), torch.empty(2, 5, 0, device=gpu), torch.empty(0, 4, device=gpu), B, C)
    spoil(gpu, [B.numel()] * 8)
    for g in torch.autograd.grad(y.sum(), (B, C)):
        assert torch.equal(g, torch.zeros_like(B))


@pytest.mark.parametrize("quant", [torch.int8, torch.float8_e4m3fn])
def test_eight_bits_of_no_channels(gpu, quant):
    """A row without values is a row of zeros: its scale is 1."""
    x, w = torch.empty(5, 60, 0, device=gpu, dtype=torch.bfloat16), torch.empty(0, device=gpu)
    spoil(gpu, [300] * 8)
    q, scale = f.rms_norm(x, w, quant=quant)
    assert q.shape == x.shape and torch.equal(scale, torch.ones(5, 60, device=gpu))
    spoil(gpu, [300] * 8)
    q, scale, total = f.rms_norm(x, w, x.float(), quant=quant)
    assert total.shape == x.shape and torch.equal(scale, torch.ones(5, 60, device=gpu))


def test_sums_over_many_parts_are_no_long_chains(gpu):
    """A parameter's gradient is joined from 65 536 stretches of 128 tokens here. Positive values that are all alike round the same way
    every time; a path to the result has at most 128 additions of tokens and two levels of 64 + 16 of stretches, each of which
    rounds by half a unit in the last place, 2^-24, of a partial sum that is no larger than the whole."""
    batch, T, value = 64, 131072, 1.990972876548767
    x = torch.ones(batch, T, 8, device=gpu)
    w, b = torch.randn(8, 4, device=gpu, requires_grad=True), torch.randn(8, device=gpu, requires_grad=True)
    gw, gb = torch.autograd.grad(f.causal_conv(x, w, b), (w, b), torch.full_like(x, value))
    value = float(torch.tensor(value))  # (as float32 holds it)
    bound = (128 + 2 * (64 + 16)) * 2.0 ** -24
    for k in range(4):  # (tap k reads no token for the first 3 - k)
        want = value * batch * (T - (3 - k))
        assert (gw[:, k].double() - want).abs().max() <= bound * want, k
    want = value * batch * T
    assert (gb.double() - want).abs().max() <= bound * want


def test_selective_scan_of_many_sequences(gpu):
    """65 536 sequences of one token: with h[-1] = 0, y = x (d (B . C) + D), and gradients that follow from that. Roundings of 2^-24: some
    64 (softplus, products, sums over 16 states), for the gradients of B and C those of sums over channels (32 of a block, 64 blocks), for D's
    those of sums over 65 536 parts in two levels, all of the sum of the terms' sizes; and one to bfloat16."""
    S, D, N = 65536, 2048, 16
    g = torch.Generator(device=gpu).manual_seed(1)
    r = lambda *s: torch.randn(s, generator=g, device=gpu)  # noqa: E731
    x, dt, gy = (r(S, 1, D).to(torch.bfloat16) for _ in range(3))
    B, C = (r(S, 1, N).to(torch.bfloat16) for _ in range(2))
    A, skip = -r(D, N).exp(), r(D)
    leaves = [t.requires_grad_() for t in (x, dt, A, B, C, skip)]
    y = f.selective_scan(*leaves, softplus=True)
    gx, gdt, gA, gB, gC, gskip = torch.autograd.grad(y, leaves, gy)
    assert torch.equal(gA, torch.zeros_like(A))
    some = torch.tensor([0, 1, 7, 4095, 32767, 65007, 65024, 65025, 65535], device=gpu)  # (a launch's last parts and the next one's first among them)
    with torch.no_grad():
        w = {k: t[some, 0].double() for k, t in dict(x=x, dt=dt, gy=gy, B=B, C=C).items()}
        d, mixed = torch.nn.functional.softplus(w["dt"], threshold=60.0), (w["B"] * w["C"]).sum(-1, keepdim=True)
        terms = w["gy"] * d * w["x"]
        along, whole = terms.sum(-1, keepdim=True), terms.abs().sum(-1, keepdim=True)
        want = {"y": w["x"] * (d * mixed + skip.double()), "gx": w["gy"] * (d * mixed + skip.double()),
                "gdt": w["gy"] * w["x"] * mixed * torch.sigmoid(w["dt"]), "gB": along * w["C"], "gC": along * w["B"]}
        for name, got in (("y", y), ("gx", gx), ("gdt", gdt), ("gB", gB), ("gC", gC)):
            got, ref = got[some, 0].double(), want[name]
            size = whole * {"gB": w["C"], "gC": w["B"]}[name].abs() if name in ("gB", "gC") else ref.abs().max()
            assert ((got - ref).abs() <= 2.0 ** -8 * 1.01 * ref.abs() + (64 + D // 16) * 2.0 ** -24 * size).all(), name
        ref, size = torch.zeros(D, dtype=torch.float64, device=gpu), torch.zeros(D, dtype=torch.float64, device=gpu)
        for a, b in zip(x.split(8192), gy.split(8192)):
            part = a[:, 0].double() * b[:, 0].double()
            ref, size = ref + part.sum(0), size + part.abs().sum(0)
        assert ((gskip.double() - ref).abs() <= (16 + 2 * 80) * 2.0 ** -24 * size).all()


def test_selective_scan_of_many_tokens_and_states(gpu):
    """131 073 sequences of 64 tokens with 256 states: 2^31 values of B and C and more, numbered with more than 32 bits backwards."""
    S, T, D, N = 131073, 64, 4, 256
    g = torch.Generator(device=gpu).manual_seed(2)
    r = lambda *s: torch.randn(s, generator=g, device=gpu)  # noqa: E731
    x, dt, gy = r(S, T, D).to(torch.bfloat16), (r(S, T, D) - 2).to(torch.bfloat16), r(S, T, D).to(torch.bfloat16)
    B, C = (torch.empty(S, T, N, dtype=torch.bfloat16, device=gpu).normal_(generator=g) for _ in range(2))
    A = -r(D, N).exp()
    leaves = [t.requires_grad_() for t in (x, dt, A, B, C)]
    y = f.selective_scan(*leaves, softplus=True)
    gx, gdt, gA, gB, gC = torch.autograd.grad(y, leaves, gy)
    some = [0, 65535, 65536, 131072]
    ref = [t.detach()[some].cpu().double().requires_grad_() if t is not A else A.detach().cpu().double().requires_grad_() for t in leaves]
    want = baseline.naive_selective_scan(*ref, softplus=True)
    wants = torch.autograd.grad(want, [ref[i] for i in (0, 1, 3, 4)], gy[some].cpu().double())
    for name, got, w in (("y", y, want), ("gx", gx, wants[0]), ("gdt", gdt, wants[1]), ("gB", gB, wants[2]), ("gC", gC, wants[3])):
        got, w = got.detach()[some].cpu().double(), w.detach()
        bound = 2.0 ** -8 * 1.01 * w.abs() + (64 + 2 * T) * 2.0 ** -24 * w.abs().max()
        assert ((got - w).abs() <= bound).all(), name
    assert torch.isfinite(gA).all()


def test_selective_scan_of_many_groups(gpu):
    """A group a channel, more of them than a grid's second dimension holds workgroups."""
    D = 70000
    g = torch.Generator(device=gpu).manual_seed(3)
    x, dt, B, C, gy = (torch.randn(1, 3, D, generator=g, device=gpu) for _ in range(5))
    A = -torch.randn(D, 1, generator=g, device=gpu).exp()
    leaves = [t.requires_grad_() for t in (x, dt, A, B[..., None], C[..., None])]
    y = f.selective_scan(*leaves, softplus=True)
    grads = torch.autograd.grad(y, leaves, gy)
    ref = [t.detach().cpu().double().requires_grad_() for t in leaves]
    want = baseline.naive_selective_scan(*ref, softplus=True)
    for got, w in zip([y, *grads], [want, *torch.autograd.grad(want, ref, gy.cpu().double())]):
        got, w = got.detach().cpu().double(), w.detach()
        assert ((got - w).abs() <= 2.0 ** -24 * w.abs() + (64 + 2 * 3) * 2.0 ** -24 * w.abs().max()).all()


@pytest.mark.parametrize("native", [True, False])
def test_a_single_token_stored_time_first(gpu, monkeypatch, native):
    """[batch, 1, channels] as a view of [1, batch, channels]: where the next token would be is far away, and does not matter."""
    if not native:
        monkeypatch.setattr(state_space, "_native", None)
    S, D, N = 4096, 1024, 4
    g = torch.Generator(device=gpu).manual_seed(4)
    first = [torch.randn(1, S, D, generator=g, device=gpu).transpose(0, 1) for _ in range(4)]
    B, C = (torch.randn(1, S, N, generator=g, device=gpu).transpose(0, 1) for _ in range(2))
    A = -torch.randn(D, N, generator=g, device=gpu).exp()
    assert first[0].stride(1) == 1 << 22
    results = []
    for lay in (lambda t: t, lambda t: t[:, 0].clone()[:, None]):
        x, dt, z, gy, b, c = (lay(t) for t in (*first, B, C))
        leaves = [t.detach().requires_grad_() for t in (x, dt, A, b, c, z)]
        y = f.selective_scan(leaves[0], leaves[1], leaves[2], leaves[3], leaves[4], z=leaves[5], softplus=True)
        results.append([y, *torch.autograd.grad(y, leaves, gy)])
    assert all(torch.equal(p, q) for p, q in zip(*results))


def test_selections_of_far_tokens(gpu):
    """16 384 groups with 256 states: 2^22 values of B a token, more than the kernels reach over within a tile."""
    G, N = 16384, 256
    g = torch.Generator(device=gpu).manual_seed(5)
    x, dt, gy = (torch.randn(1, 3, G, generator=g, device=gpu) for _ in range(3))
    B, C = (torch.randn(1, 3, G, N, generator=g, device=gpu) for _ in range(2))
    A = -torch.randn(G, N, generator=g, device=gpu).exp()
    leaves = [t.requires_grad_() for t in (x, dt, A, B, C)]
    y = f.selective_scan(*leaves, softplus=True)
    grads = torch.autograd.grad(y, leaves, gy)
    ref = [t.detach().cpu().double().requires_grad_() for t in leaves]
    want = baseline.naive_selective_scan(*ref, softplus=True)
    for got, w in zip([y, *grads], [want, *torch.autograd.grad(want, ref, gy.cpu().double())]):
        got, w = got.detach().cpu().double(), w.detach()
        assert got.shape == w.shape and ((got - w).abs() <= 2.0 ** -24 * w.abs() + (64 + 2 * 3) * 2.0 ** -24 * w.abs().max()).all()


@pytest.mark.parametrize("quant", [None, torch.float8_e4m3fn])
def test_norm_of_many_rows(gpu, quant):
    """More rows than a launch has waves for, of a width at which rows begin inside vectors: every row is its own norm."""
    rows, D = (1 << 26) + 3, 9
    g = torch.Generator(device=gpu).manual_seed(6)
    x = torch.empty(rows, D, dtype=torch.bfloat16, device=gpu).normal_(generator=g)
    r = torch.empty(rows, D, dtype=torch.bfloat16, device=gpu).normal_(generator=g)
    w = torch.randn(D, generator=g, device=gpu)
    outs = f.rms_norm(x, w, r, quant=quant)
    if quant is None:
        leaves = [t.clone().requires_grad_() for t in (x, w, r)]
        gx, gw, _ = torch.autograd.grad(f.rms_norm(*leaves)[0], leaves, x)
        assert torch.isfinite(gw).all()
    for start in range(0, rows, 1 << 23):  # (each piece is a call of one launch)
        piece = slice(start, min(rows, start + (1 << 23)))
        want = f.rms_norm(x[piece], w, r[piece], quant=quant)
        for got, one in zip(outs, want):
            assert torch.equal(got[piece].view(torch.uint8), one.view(torch.uint8)), start
    last = slice(rows - 5, rows)
    total = (x[last].float() + r[last].float()).to(torch.bfloat16)
    assert torch.equal(outs[-1][last], total)
    if quant is None:
        leaf, wide = total.double().requires_grad_(), w.double()
        y = leaf / torch.sqrt(leaf.square().mean(-1, keepdim=True) + 1e-6) * wide
        (want,) = torch.autograd.grad(y, leaf, x[last].double())
        for got, one in ((outs[0][last], y.detach()), (gx[last], want)):
            assert ((got.double() - one).abs() <= 2.0 ** -8 * 1.01 * one.abs() + 64 * 2.0 ** -24 * one.abs().max()).all()


def test_convolution_of_many_sequences(gpu):
    """More sequences than a launch has lanes for, one token each: y = w[1] x + w[0] state, and gradients that follow from that. Roundings of
    2^-24: 3 of an output; 3 x 80 + 16 of a parameter's gradient (8 388 617 parts in three levels)."""
    S, D = (1 << 23) + 9, 4
    g = torch.Generator(device=gpu).manual_seed(7)
    x, gy, kept, gkept = (torch.randn(S, 1, D, generator=g, device=gpu) for _ in range(4))
    w = torch.randn(D, 2, generator=g, device=gpu)
    leaves = [t.requires_grad_() for t in (x, w, kept)]
    y, new = f.causal_conv(leaves[0], leaves[1], state=leaves[2], return_state=True)
    assert torch.equal(new, x)
    gx, gw, gstate = torch.autograd.grad((y, new), leaves, (gy, gkept))
    with torch.no_grad():
        a, b = w[:, 1].double(), w[:, 0].double()
        for start in range(0, S, 1 << 21):
            p = slice(start, start + (1 << 21))
            for got, terms in ((y, (a * x[p], b * kept[p])), (gx, (a * gy[p], gkept[p].double())), (gstate, (b * gy[p],))):
                assert ((got[p] - sum(terms)).abs() <= 3 * 2.0 ** -24 * sum(t.abs() for t in terms)).all()
        for k, rows in ((0, kept), (1, x)):
            terms = gy.double() * rows
            assert ((gw[:, k] - terms.sum((0, 1))).abs() <= (16 + 3 * 80) * 2.0 ** -24 * terms.abs().sum((0, 1))).all()


@pytest.mark.parametrize("rows,D,N", [((1 << 24) + 5, 4, 1), (2, 1 << 20, 128)])
def test_steps_of_many_rows_or_channels(gpu, rows, D, N):
    """More than a launch has threads or a grid's second dimension workgroups for: the rows and channels of calls of their own."""
    g = torch.Generator(device=gpu).manual_seed(8)
    x, dt = (torch.randn(rows, D, generator=g, device=gpu) for _ in range(2))
    B, C = (torch.randn(rows, N, generator=g, device=gpu) for _ in range(2))
    A, state = -torch.rand(D, N, generator=g, device=gpu), torch.randn(rows, D, N, generator=g, device=gpu)
    kept, w = torch.randn(rows, 2, D, generator=g, device=gpu), torch.randn(D, 3, generator=g, device=gpu)
    slots = torch.randperm(rows, generator=g, device=gpu)
    new, new_kept = state.clone(), kept.clone()
    y, u = f.selective_scan_step(new, x, dt, A, B, C, softplus=True, slots=slots), f.causal_conv_step(new_kept, x, w, slots=slots)
    for r in (slice(0, min(rows, 9)), slice(max(0, rows - 9), rows)):
        for c in (slice(0, min(D, 64)), slice(D - min(D, 64), D)):
            mine = slots[r]
            one, one_kept = state[mine][:, c].contiguous(), kept[mine][..., c].contiguous()
            assert torch.equal(f.selective_scan_step(one, x[r, c], dt[r, c], A[c], B[r], C[r], softplus=True), y[r, c]) and torch.equal(new[mine][:, c], one)
            assert torch.equal(f.causal_conv_step(one_kept, x[r, c], w[c]), u[r, c]) and torch.equal(new_kept[mine][..., c], one_kept)


@pytest.mark.parametrize("native", [True, False])
def test_what_is_too_large_is_named(gpu, monkeypatch, native):
    """Sizes that no call takes, of expanded tensors that hold one value: refused by name before anything is allocated."""
    if not native:
        monkeypatch.setattr(state_space, "_native", None)
    one = torch.ones(1, device=gpu)
    many, wide = 1 << 31, (1 << 20) + 16
    for call in (lambda: f.rms_norm(one.expand(many, 1), one),
                 lambda: f.causal_conv(one.expand(1, many, 1), one[None]), lambda: f.causal_conv(one.expand(2, many // 2, 1), one[None]),
                 lambda: f.causal_conv(one.expand(1, 1, wide), one[None].expand(wide, 1)),
                 lambda: f.causal_conv_step(torch.empty(1, 0, 1, device=gpu).expand(many, 0, 1).contiguous(), one.expand(many, 1), one[None]),
                 lambda: f.selective_scan(one.expand(1, many, 1), one.expand(1, many, 1), one[None], one.expand(1, many, 1), one.expand(1, many, 1)),
                 lambda: f.selective_scan(one.expand(1, 1, wide), one.expand(1, 1, wide), one[None].expand(wide, 1), one.expand(1, 1, 1), one.expand(1, 1, 1)),
                 lambda: f.selective_scan_step(torch.ones(1, 1, 1, device=gpu), one.expand(many, 1), one.expand(many, 1), one[None], one.expand(many, 1), one.expand(many, 1),
                                               slots=torch.zeros(1, dtype=torch.int32, device=gpu).expand(many))):
        before = torch.cuda.memory_allocated()
        with pytest.raises(AssertionError, match="a call takes up to"):
            call()
        assert torch.cuda.memory_allocated() == before


@pytest.mark.parametrize("quant,limit", [(torch.int8, 127.0), (torch.float8_e4m3fn, 448.0)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("residual", [None, "same", torch.float32])
@pytest.mark.parametrize("D", [2047, 2049, 2500])
def test_eight_bits_of_many_rows(gpu, quant, limit, dtype, residual, D):
    """A wave a row, several vectors a lane, rows that begin inside a vector (or not), of a number that is no multiple of a workgroup's. q stands for
    y to half a step of its type (1/2 for integers; a 16th of the value, or 2^-10, for floats), after three roundings of 2^-24, and a
    row that holds a NaN or an infinity has neither values nor a scale."""
    rows = 1030
    g = torch.Generator(device=gpu).manual_seed(9)
    x, w = torch.randn(rows, D, generator=g, device=gpu).to(dtype), 1 + 0.2 * torch.randn(D, generator=g, device=gpu)
    r = None if residual is None else (3 * torch.randn(rows, D, generator=g, device=gpu)).to(dtype if residual == "same" else residual)
    x[7], x[11, 0], x[12, D - 1], x[1029, D // 2] = 0, float("nan"), float("inf"), float("-inf")
    if r is not None:
        r[7] = 0
    total = x if r is None else (x.float() + r.float()).to(r.dtype)
    q, scale, *more = f.rms_norm(x, w, r, eps=1e-5, quant=quant)
    if r is not None:
        assert torch.equal(more[0].isnan(), total.isnan()) and torch.equal(more[0].nan_to_num(), total.nan_to_num())
    lost = torch.zeros(rows, dtype=torch.bool, device=gpu)
    lost[[11, 12, 1029]] = True
    assert torch.equal(scale.isnan(), lost)
    if quant == torch.int8:
        assert (q[lost] == 0).all()
    else:
        assert torch.equal(q.float().isnan().all(1), lost) and torch.equal(q.float().isnan().any(1), lost)
    wide = total[~lost].double()
    want = wide / torch.sqrt(wide.square().mean(-1, keepdim=True) + 1e-5) * w.double()
    q, scale = q[~lost].double(), scale[~lost].double().unsqueeze(-1)
    most = want.abs().amax(-1, keepdim=True)
    assert ((scale - torch.where(most == 0, 1.0, most / limit)).abs() <= 64 * 2.0 ** -24 * scale).all()
    step = torch.full_like(want, 0.5) if quant == torch.int8 else torch.maximum(want.abs() / scale / 16, torch.full_like(want, 2.0 ** -10))
    assert ((q * scale - want).abs() <= step * scale * (1 + 1e-4)).all()
    assert (q[want == 0] == 0).all() and (q.abs().amax(-1) == torch.where(most[:, 0] == 0, 0.0, limit)).all()
