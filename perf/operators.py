"""
The operators of a state space layer in a language model, as cases that can be timed and compared.

  scan   ``selective_scan`` over whole prompts (``mode`` "prompt"), with its gradients ("train"), and
         ``selective_scan_step`` for one token of each sequence ("step")
  conv   ``causal_conv`` and ``causal_conv_step``, the short convolution before the scan, in the same modes
  norm   ``rms_norm`` with the residual's addition: "train" with gradients, "prompt" with an output in 8 bits

Fields of a case besides ``op`` and ``mode``: ``dtype`` (of the activations; parameters and states are float32),
``batch`` and ``T`` (the tokens; a step's ``batch`` is the sequences that take one token), ``D`` channels, and

  scan   ``N`` states a channel, ``groups`` of channels that share B and C, ``gate`` (z is given)
  conv   ``K`` taps
  both   ``packed`` (``batch`` sequences of different lengths, some of them empty, behind each other in ``batch * T``
         tokens), ``state`` (prompts: a state is handed in and the new one handed back)
  norm   ``residual`` (its type), ``eight`` ("" or the type of the 8-bit output)

``own`` is set from outside: false computes the plain form in 32 bits, true calls the framework.
"""
import math

import numpy as np
import torch

own = False

_TYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16, "int8": torch.int8,
          "float8": torch.float8_e4m3fn}
_SIZE = {"float32": 4, "bfloat16": 2, "float16": 2, "int8": 1, "float8": 1}
_EPS = 1e-5


def _scan(name, mode, dtype, batch, T, D, N=16, groups=1, gate=True, packed=False, state=False):
    return {"name": name, "op": "scan", "mode": mode, "dtype": dtype, "batch": batch, "T": T, "D": D, "N": N,
            "groups": groups, "gate": gate, "packed": packed, "state": state}


def _conv(name, mode, dtype, batch, T, D, K=4, packed=False, state=False):
    return {"name": name, "op": "conv", "mode": mode, "dtype": dtype, "batch": batch, "T": T, "D": D, "K": K,
            "packed": packed, "state": state}


def _norm(name, mode, dtype, batch, T, D, residual="", eight=""):
    return {"name": name, "op": "norm", "mode": mode, "dtype": dtype, "batch": batch, "T": T, "D": D,
            "residual": residual, "eight": eight}


def listed():
    return [
        # One token of one user's answer: the call itself is all there is.
        _scan("scan_step_one", "step", "bfloat16", 1, 1, 2048),
        # One token of each of many answers that are served together.
        _scan("scan_step_many", "step", "bfloat16", 512, 1, 2048),
        # A short prompt in float32, of an odd length, to a small model.
        _scan("scan_prompt_short", "prompt", "float32", 1, 173, 512, state=True),
        # Prompts of different lengths behind each other, as a server takes them in.
        _scan("scan_prompts_packed", "prompt", "bfloat16", 13, 617, 2048, packed=True, state=True),
        # One long document, few channels: there is more time than there are channels.
        _scan("scan_long_train", "train", "float32", 1, 30001, 256),
        # A training step of the large layer at training batch size.
        _scan("scan_layer_train", "train", "bfloat16", 8, 4096, 2048),
        # The convolution's part of a token of each of many answers.
        _conv("conv_step_many", "step", "bfloat16", 512, 1, 2048),
        # ... of the packed prompts.
        _conv("conv_prompts_packed", "prompt", "bfloat16", 13, 617, 2048, packed=True, state=True),
        # ... of the training step.
        _conv("conv_layer_train", "train", "bfloat16", 8, 4096, 2048),
        # The norm before a served token's projections in 8 bits.
        _norm("norm_token_float8", "prompt", "bfloat16", 16, 1, 2048, "bfloat16", "float8"),
        # ... before those of a prompt, at a width that is no whole number of vectors.
        _norm("norm_prompt_float8", "prompt", "bfloat16", 8, 2048, 2049, "bfloat16", "float8"),
        # The norm of the training step, its residual stream kept in float32.
        _norm("norm_layer_train", "train", "bfloat16", 8, 4096, 2048, "float32"),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi))))))))


# The most states (tokens x D x N) and values (tokens x D) of one drawn call: the listed layers'.
_MOST_STATES, _MOST_VALUES = 1 << 30, 1 << 26


def draw(rng):
    op = rng.choices(("scan", "conv", "norm"), (0.5, 0.25, 0.25))[0]
    dtype = rng.choices(("float32", "bfloat16", "float16"), (0.3, 0.5, 0.2))[0]
    D = _log_int(rng, 24, 2560)
    if rng.random() < 0.6:  # the widths that models choose
        D = max(32, D - D % 32)
    if op == "norm":
        mode = rng.choice(("prompt", "train"))
        rows = _log_int(rng, 1, _MOST_VALUES // D)
        batch = _log_int(rng, 1, min(rows, 64))
        return {k: v for k, v in _norm("", mode, dtype, batch, max(1, rows // batch), D, rng.choice(("", dtype, "float32")),
                                       rng.choice(("int8", "float8")) if mode == "prompt" else "").items() if k != "name"}
    mode = rng.choices(("step", "prompt", "train"), (0.25, 0.4, 0.35))[0]
    N = rng.choice((8, 16, 16, 16, 32, 64)) if rng.random() < 0.8 else _log_int(rng, 1, 128)
    most = min(_MOST_VALUES // D, _MOST_STATES // (D * N)) if op == "scan" else _MOST_VALUES // D
    if mode == "step":
        batch, T = _log_int(rng, 1, min(1024, most)), 1
    else:
        tokens = _log_int(rng, 16, most)
        batch = _log_int(rng, 1, min(64, tokens))
        T = min(32768, max(1, tokens // batch))
    packed = mode != "step" and batch > 1 and rng.random() < 0.4
    state = mode == "prompt" and rng.random() < 0.6
    if op == "conv":
        case = _conv("", mode, dtype, batch, T, D, rng.choice((2, 3, 4, 4, 4, 8)), packed, state)
    else:
        groups = rng.choice([1, 1, 1] + [g for g in (2, 4, 8) if D % g == 0 and D // g >= 16])
        case = _scan("", mode, dtype, batch, T, D, N, groups, rng.random() < 0.7, packed, state)
    del case["name"]
    return case


def _lengths(case, seed):
    """Lengths of ``batch`` sequences, ``batch * T`` tokens in all: of any ratio to each other, about one in ten empty."""
    r = np.random.default_rng(seed)
    share = r.lognormal(0.0, 1.0, case["batch"]) * (r.random(case["batch"]) > 0.1)
    share[r.integers(case["batch"])] += 0.5
    ends = np.round(np.cumsum(share) / share.sum() * (case["batch"] * case["T"])).astype(np.int64)
    ends[-1] = case["batch"] * case["T"]
    return np.diff(ends, prepend=0)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype, D, train, step = _TYPES[case["dtype"]], case["D"], case["mode"] == "train", case["mode"] == "step"
    packed = case.get("packed", False)
    lead = (1, case["batch"] * case["T"]) if packed else (case["batch"], case["T"])
    if step:
        lead = (case["batch"],)

    def normal(*shape, of=dtype, scale=1.0, at=0.0):
        return torch.randn(shape, generator=gen, device="cuda").mul_(scale).add_(at).to(of)

    def leaf(t):
        return t.detach().requires_grad_(train)

    s = {"case": case}
    if case["op"] == "norm":
        s["x"] = leaf(normal(*lead, D))
        s["weight"] = leaf(normal(D, of=torch.float32, scale=0.1, at=1.0))
        if case["residual"]:
            s["residual"] = leaf(normal(*lead, D, of=_TYPES[case["residual"]], scale=2.0))
        if train:
            s["grad"] = normal(*lead, D)
            s["residual_grad"] = normal(*lead, D, of=_TYPES[case["residual"]]) if case["residual"] else None
        return s
    sequences, slots = case["batch"], case["batch"] + 3  # (steps: more states are kept than take a token)
    if packed:
        s["offsets"] = torch.from_numpy(np.concatenate([[0], np.cumsum(_lengths(case, seed))]).astype(np.int32)).cuda()
    if step:
        s["slots"] = torch.randperm(slots, generator=gen, device="cuda")[:sequences].to(torch.int32)
    if case["op"] == "conv":
        K = case["K"]
        # (the convolution's input is the first half of the projection that gives the gate as well)
        s["x"] = leaf(normal(*lead, 2 * D)[..., :D])
        s["weight"] = leaf(normal(D, K, of=torch.float32, scale=K ** -0.5))
        s["bias"] = leaf(normal(D, of=torch.float32, scale=0.1))
        if step or case["state"]:
            s["state"] = normal(slots if step else sequences, K - 1, D)
    else:
        N, G = case["N"], case["groups"]
        s["x"] = leaf(normal(*lead, D))
        s["dt"] = leaf(normal(*lead, D, scale=0.5))
        s["A"] = leaf(normal(D, N, of=torch.float32, scale=0.1).exp_().mul_(-torch.arange(1, N + 1, device="cuda")))
        # (B and C are parts of one projection, the gate the second half of the layer's first one)
        parts = normal(*lead, 8 + 2 * G * N)
        s["B"], s["C"] = (leaf(parts[..., a:a + G * N].unflatten(-1, (G, N))) for a in (8, 8 + G * N))
        s["D"] = leaf(normal(D, of=torch.float32, scale=0.1, at=1.0))
        s["z"] = leaf(normal(*lead, 2 * D)[..., D:]) if case["gate"] else None
        steps = torch.rand(D, generator=gen, device="cuda").mul_(math.log(100.0)).add_(math.log(1e-3)).exp_()
        s["dt_bias"] = leaf(steps.expm1().log())  # softplus gives step sizes of 0.001 to 0.1
        if step or case["state"]:
            s["state"] = normal(slots if step else sequences, D, N, of=torch.float32)
    if train:
        s["grad"] = normal(*lead, D)
    return s


def run(s):
    case = s["case"]
    if own:
        return _run_own(case, s)
    with torch.no_grad():
        return {"scan": _plain_scan, "conv": _plain_conv, "norm": _plain_norm}[case["op"]](case, s)


# ---------------------------------------------------------------------------------------------- the framework's calls
def _run_own(case, s):
    import scanscam_amd as f

    op, mode = case["op"], case["mode"]
    if op == "norm":
        names = ["x", "weight"] + (["residual"] if case["residual"] else [])
        if mode == "prompt":
            got = f.rms_norm(s["x"], s["weight"], s.get("residual"), eps=_EPS, quant=_TYPES[case["eight"]])
            return _norm_outputs(case, *got)
        got = f.rms_norm(s["x"], s["weight"], s.get("residual"), eps=_EPS)
        out, grads = ((got,), (s["grad"],)) if not case["residual"] else (got, (s["grad"], s["residual_grad"]))
        back = torch.autograd.grad(out, [s[n] for n in names], grads)
        return _named(("out", "sum"), out) | _named(names, back, "_grad")
    if op == "conv":
        names = ["x", "weight", "bias"]
        if mode == "step":
            out = f.causal_conv_step(s["state"], s["x"], s["weight"], s["bias"], activation="silu", slots=s["slots"])
            return {"out": out, "state": s["state"]}
        got = f.causal_conv(s["x"], s["weight"], s["bias"], activation="silu", state=s.get("state"),
                            offsets=s.get("offsets"), return_state=case["state"])
    else:
        names = ["x", "dt", "A", "B", "C", "D", "dt_bias"] + (["z"] if case["gate"] else [])
        given = [s[n] for n in ("x", "dt", "A", "B", "C", "D", "z", "dt_bias")]
        if mode == "step":
            out = f.selective_scan_step(s["state"], *given, softplus=True, slots=s["slots"])
            return {"out": out, "state": s["state"]}
        got = f.selective_scan(*given, softplus=True, state=s.get("state"), offsets=s.get("offsets"),
                               return_state=case["state"])
    if mode == "prompt":
        return {"out": got[0], "state": got[1]} if case["state"] else {"out": got}
    return {"out": got.detach()} | _named(names, torch.autograd.grad(got, [s[n] for n in names], s["grad"]), "_grad")


def _named(names, values, ending=""):
    return {n + ending: v.detach() for n, v in zip(names, values)}


def _norm_outputs(case, q, scale, total=None):
    """What a norm in 8 bits hands over; integers as the values that they stand for."""
    if case["eight"] == "int8":
        q = (q * scale.unsqueeze(-1)).to(torch.bfloat16)
    return {"out": q, "scale": scale} | ({} if total is None else {"sum": total})


# ------------------------------------------------------------------------------------------------------- plain forms
def _sequences(case, s):
    """For the tokens of all sequences behind each other: the sequence of each, its place there and the sequence's length."""
    tokens = case["batch"] * case["T"]
    at = torch.arange(tokens, device="cuda")
    if "offsets" not in s:
        return at // case["T"], at % case["T"], torch.full_like(at, case["T"])
    offsets = s["offsets"].long()
    of = torch.bucketize(at, offsets[1:], right=True)
    return of, at - offsets[of], (offsets[1:] - offsets[:-1])[of]


def _recurrence(a, b):
    """h[t] = a[t] h[t-1] + b[t] along the first dimension, spans doubled."""
    span = 1
    while span < a.shape[0]:
        b = torch.cat((b[:span], torch.addcmul(b[span:], a[span:], b[:-span])))
        a = torch.cat((a[:span], a[span:] * a[:-span]))
        span *= 2
    return b


def _plain_scan(case, s):
    D, N, G, dtype = case["D"], case["N"], case["groups"], _TYPES[case["dtype"]]
    x, dt, z = (None if s[k] is None else s[k].float().reshape(-1, D) for k in ("x", "dt", "z"))
    B, C = (s[k].float().reshape(-1, G, 1, N) for k in ("B", "C"))
    A, shape = s["A"].view(G, D // G, N), s["x"].shape
    raw = dt + s["dt_bias"]
    dt = torch.maximum(raw, torch.zeros_like(raw)) + torch.log1p(torch.exp(-raw.abs()))
    split = lambda v: v.view(-1, G, D // G, 1)  # noqa: E731
    decay = torch.exp(split(dt) * A)
    into = split(dt * x) * B
    kept = {}
    if case["mode"] == "step":
        slots = s["slots"].long()
        h = decay * s["state"][slots].view(decay.shape) + into
        s["state"][slots] = h.view(-1, D, N)
        kept = {"state": s["state"]}
    else:
        of, place, length = _sequences(case, s)
        first = (place == 0).view(-1, 1, 1, 1)
        if case["state"]:
            into = into + torch.where(first, decay * s["state"].view(-1, *decay.shape[1:])[of], 0.0)
        decay = torch.where(first, 0.0, decay)
        h = _recurrence(decay, into)
        if case["state"]:
            new = s["state"].clone()
            last = place == length - 1
            new[of[last]] = h[last].view(-1, D, N)
            kept = {"state": new}
    del into
    ungated = (h * C).sum(-1).view(-1, D) + s["D"] * x
    sigmoid = None if z is None else 1.0 / (1.0 + torch.exp(-z))
    out = ungated if z is None else ungated * (z * sigmoid)
    kept["out"] = out.to(dtype).view(shape)
    if case["mode"] != "train":
        return kept
    grad = s["grad"].float().reshape(-1, D)
    if z is not None:
        kept["z_grad"] = (grad * ungated * sigmoid * (1.0 + z * (1.0 - sigmoid))).to(dtype).view(shape)
        grad = grad * (z * sigmoid)
    later = torch.cat((decay[1:], torch.zeros_like(decay[:1])))
    g = _recurrence(later.flip(0), (split(grad) * C).flip(0)).flip(0)
    del later
    kept["C_grad"] = (split(grad) * h).sum(2).to(dtype).view(s["C"].shape)
    kept["B_grad"] = (split(dt * x) * g).sum(2).to(dtype).view(s["B"].shape)
    along = (g * B).sum(-1).view(-1, D)
    q = g * decay
    q[1:] *= h[:-1]
    q[0] = 0.0
    dt_grad = (x * along + (q * A).sum(-1).view(-1, D)) / (1.0 + torch.exp(-raw))
    kept["A_grad"] = (q * split(dt)).sum(0).view(D, N)
    kept["x_grad"] = (dt * along + s["D"] * grad).to(dtype).view(shape)
    kept["dt_grad"] = dt_grad.to(dtype).view(shape)
    kept["dt_bias_grad"] = dt_grad.sum(0)
    kept["D_grad"] = (grad * x).sum(0)
    return kept


def _plain_conv(case, s):
    D, K, dtype, shape = case["D"], case["K"], _TYPES[case["dtype"]], s["x"].shape
    x, taps = s["x"].float().reshape(-1, D), s["weight"].t().contiguous()
    back = torch.arange(K - 1, -1, -1, device="cuda")  # tap k reads so many tokens back
    kept = {}
    if case["mode"] == "step":
        slots = s["slots"].long()
        window = torch.cat((s["state"][slots].float(), x.unsqueeze(1)), dim=1)
        s["state"][slots] = window[:, 1:].to(dtype)
        kept["state"] = s["state"]
    else:
        of, place, length = _sequences(case, s)
        # All rows that a tap can read: the states', the tokens', and one of zeros.
        before = s["state"].float().view(-1, D) if case["state"] else x[:0]
        rows = torch.cat((before, x, torch.zeros_like(x[:1])))
        at = torch.arange(x.shape[0], device="cuda")

        def taken(token, seq, spot, count):
            inside, ahead = before.shape[0] + token - count, seq * (K - 1) + (K - 1) + spot - count
            return torch.where(spot >= count, inside, ahead if case["state"] else torch.full_like(inside, -1) + rows.shape[0])

        index = taken(at[:, None], of[:, None], place[:, None], back)
        window = rows[index]
        if case["state"]:
            each = torch.arange(case["batch"], device="cuda")
            ends = s["offsets"].long() if case["packed"] else torch.arange(case["batch"] + 1, device="cuda") * case["T"]
            kept["state"] = rows[taken(ends[1:, None], each[:, None], (ends[1:] - ends[:-1])[:, None], back[:-1])].to(dtype)
    p = (window * taps).sum(1) + s["bias"]
    sigmoid = 1.0 / (1.0 + torch.exp(-p))
    kept["out"] = (p * sigmoid).to(dtype).view(shape)
    if case["mode"] != "train":
        return kept
    grad = s["grad"].float().reshape(-1, D) * sigmoid * (1.0 + p * (1.0 - sigmoid))
    kept["weight_grad"] = (window * grad.unsqueeze(1)).sum(0).t().contiguous()
    kept["bias_grad"] = grad.sum(0)
    del window
    grads = torch.cat((grad, torch.zeros_like(grad[:1])))
    onto = torch.where((place[:, None] + back) < length[:, None], at[:, None] + back, x.shape[0])
    kept["x_grad"] = (grads[onto] * taps).sum(1).to(dtype).view(shape)
    return kept


def _plain_norm(case, s):
    # The sum as it is stored is what is normalised, so that the gradient is that of what was computed.
    total = None if not case["residual"] else (s["x"].float() + s["residual"].float()).to(s["residual"].dtype)
    r = (s["x"] if total is None else total).float()
    rstd = torch.rsqrt((r * r).mean(-1, keepdim=True) + _EPS)
    unit = r * rstd
    y = unit * s["weight"]
    if case["eight"]:
        kind = _TYPES[case["eight"]]
        limit = 127.0 if kind is torch.int8 else 448.0
        most = y.abs().amax(-1, keepdim=True)
        scale = torch.where(most == 0.0, 1.0, most / limit)
        q = (y / scale).clamp(-limit, limit)
        return _norm_outputs(case, q.round().to(kind) if kind is torch.int8 else q.to(kind), scale.squeeze(-1), total)
    kept = {"out": y.to(_TYPES[case["dtype"]])}
    grad = s["grad"].float()
    u = grad * s["weight"]
    kept["weight_grad"] = (grad * unit).flatten(0, -2).sum(0)
    onto = rstd * (u - unit * (u * unit).mean(-1, keepdim=True))
    if total is not None:
        onto = onto + s["residual_grad"].float()
        kept["sum"], kept["residual_grad"] = total, onto.to(total.dtype)
    kept["x_grad"] = onto.to(s["x"].dtype)
    return kept


# ------------------------------------------------------------------------------------------------------------- cost
def work(case):
    size, D, M = _SIZE[case["dtype"]], case["D"], case["batch"] * case["T"]
    train = case["mode"] == "train"
    if case["op"] == "norm":
        r = _SIZE[case["residual"]] if case["residual"] else 0
        if train:  # x, residual -> y, sum; grads of both, sum (or x) -> grads of both
            return {"bytes": M * D * (4 * size + (4 * r if r else size)) + 16 * D, "flops": M * D * 14}
        return {"bytes": M * (D * (size + 2 * r + 1) + 4) + 4 * D, "flops": M * D * 7}
    if case["op"] == "conv":
        K = case["K"]
        kept = 0
        if case["mode"] == "step" or case["state"]:
            kept = 2 * case["batch"] * (K - 1) * D * size
        flops = M * D * (2 * K + 4)
        if train:  # x -> y; x, grad -> x's grad
            return {"bytes": M * D * 5 * size + 8 * D * (K + 1), "flops": 2 * flops + M * D * (2 * K + 8)}
        return {"bytes": M * D * 2 * size + 4 * D * (K + 1) + kept, "flops": flops}
    N, G, gate = case["N"], case["groups"], 1 if case["gate"] else 0
    kept = 2 * case["batch"] * D * N * 4 if case["mode"] == "step" or case["state"] else 0
    values = M * D * (3 + gate) + 2 * M * G * N  # x, dt, z, B, C -> y
    params = 4 * D * (N + 2)
    flops = M * D * (7 * N + 14 + 6 * gate)
    if train:  # x, dt, z, B, C, y's grad -> the grads of the first five
        return {"bytes": size * (values + M * D * (5 + 2 * gate) + 4 * M * G * N) + 2 * params,
                "flops": flops + M * D * (16 * N + 14 + 12 * gate)}
    return {"bytes": size * values + params + kept, "flops": flops}


# -------------------------------------------------------------------------------------------- the definition in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    w = {k: v.detach().double() for k, v in s.items() if isinstance(v, torch.Tensor) and v.is_floating_point()}
    if case["op"] == "norm":
        return _exact_norm(case, s, w)
    batch, D, step = case["batch"], case["D"], case["mode"] == "step"
    if step:
        bounds, which = [(i, i + 1) for i in range(batch)], s["slots"].long()
    else:
        n = _lengths(case, seed).tolist() if case["packed"] else [case["T"]] * batch
        ends = np.cumsum(n).tolist()
        bounds, which = [(e - k, e) for e, k in zip(ends, n)], torch.arange(batch, device="cuda")
    carried = step or case["state"]
    flat = {k: w[k].reshape(-1, *w[k].shape[s["x"].dim() - 1:]) for k in ("x", "dt", "z", "B", "C", "grad") if k in w}
    got = (_exact_scan if case["op"] == "scan" else _exact_conv)(case, flat, w, bounds, which, carried)
    for k in ("out", "x_grad", "dt_grad", "z_grad", "B_grad", "C_grad"):
        if k in got:
            got[k] = got[k].reshape(s["x"].shape if k == "out" else s[k[:-5]].shape)
    return got


def _exact_scan(case, flat, w, bounds, which, carried):
    D, N, G, M = case["D"], case["N"], case["groups"], flat["x"].shape[0]
    dt = torch.nn.functional.softplus(flat["dt"] + w["dt_bias"], threshold=60.0)
    x, B, C = flat["x"], flat["B"].repeat_interleave(D // G, 1), flat["C"].repeat_interleave(D // G, 1)
    if M * D * N > 1 << 27:
        B, C = flat["B"], flat["C"]  # (one group or few: expanded token by token)
    wide = (lambda v: v) if B.shape[1] == D else (lambda v: v.repeat_interleave(D // G, -2))
    train, state = case["mode"] == "train", w.get("state")
    # Sequences side by side, the longest first, so that one step serves all that have a token there.
    order = sorted(range(len(bounds)), key=lambda i: bounds[i][0] - bounds[i][1])
    starts = torch.tensor([bounds[i][0] for i in order], device="cuda")
    counts = [bounds[i][1] - bounds[i][0] for i in order]
    rows = which[torch.tensor(order, device="cuda")]
    h = state[rows].clone() if carried else torch.zeros(len(order), D, N, dtype=torch.float64, device="cuda")
    if train and (M * D * N * 8 > 40 << 30 or counts[0] > 40000):
        return None
    y = torch.empty(M, D, dtype=torch.float64, device="cuda")
    kept = torch.empty(M, D, N, dtype=torch.float64, device="cuda") if train else None
    live = len(order)
    lives = []
    for t in range(counts[0]):
        while counts[live - 1] <= t:
            live -= 1
        lives.append(live)
        i = starts[:live] + t if len(order) > 1 else slice(t, t + 1)
        d = dt[i].unsqueeze(-1)
        h[:live] = torch.exp(d * w["A"]) * h[:live] + d * x[i].unsqueeze(-1) * wide(B[i])
        y[i] = (h[:live] * wide(C[i])).sum(-1)
        if train:
            kept[i] = h[:live]
    y += w["D"] * x
    gate = torch.nn.functional.silu(flat["z"]) if case["gate"] else 1.0
    out = {"out": y * gate}
    if carried:
        state = state.clone()
        state[rows] = h
        out["state"] = state
    if not train:
        return out
    grad = flat["grad"]
    if case["gate"]:
        z = flat["z"].clone().requires_grad_()
        out["z_grad"], = torch.autograd.grad(torch.nn.functional.silu(z), z, grad * y)
    grad = grad * gate
    dB, dC = torch.zeros(2, M, G, N, dtype=torch.float64, device="cuda")
    dx, ddt = w["D"] * grad, torch.zeros_like(dt)
    dA, g = torch.zeros_like(w["A"]), torch.zeros_like(h)
    for t in range(counts[0] - 1, -1, -1):
        live = lives[t]
        i = starts[:live] + t if len(order) > 1 else slice(t, t + 1)
        d, xi, gi = dt[i].unsqueeze(-1), x[i].unsqueeze(-1), grad[i].unsqueeze(-1)
        g[:live] += gi * wide(C[i])
        dC[i] = (gi * kept[i]).view(live, G, D // G, N).sum(2)
        dB[i] = (d * xi * g[:live]).view(live, G, D // G, N).sum(2)
        along = (g[:live] * wide(B[i])).sum(-1)
        dx[i] += dt[i] * along
        g[:live] *= torch.exp(d * w["A"])
        if t > 0:
            q = g[:live] * kept[starts[:live] + t - 1 if len(order) > 1 else slice(t - 1, t)]
            dA += (q * d).sum(0)
            ddt[i] = x[i] * along + (q * w["A"]).sum(-1)
        else:
            ddt[i] = x[i] * along
    ddt *= torch.sigmoid(flat["dt"] + w["dt_bias"])
    return out | {"x_grad": dx, "dt_grad": ddt, "A_grad": dA, "B_grad": dB, "C_grad": dC, "D_grad": (grad * x).sum(0),
                  "dt_bias_grad": ddt.sum(0)}


def _exact_conv(case, flat, w, bounds, which, carried):
    D, K, state = case["D"], case["K"], w.get("state")
    train = case["mode"] == "train"
    x, weight, bias = (v.clone().requires_grad_(train) for v in (flat["x"], w["weight"], w["bias"]))
    if carried:
        state = state.clone()
    new, outs = [], []
    if case["mode"] == "step" or not case["packed"]:  # sequences of one length, together
        n = bounds[0][1] - bounds[0][0]
        ahead = state[which] if carried else torch.zeros(len(bounds), K - 1, D, dtype=torch.float64, device="cuda")
        groups = [torch.cat((ahead, x.view(len(bounds), n, D)), dim=1)]
    else:
        groups = []
        for i, (a, b) in enumerate(bounds):
            ahead = state[i] if carried else torch.zeros(K - 1, D, dtype=torch.float64, device="cuda")
            groups.append(torch.cat((ahead, x[a:b]))[None])
    for rows in groups:
        n = rows.shape[1] - (K - 1)
        p = bias
        for k in range(K):
            p = p + weight[:, k] * rows[:, k:k + n]
        outs.append(torch.nn.functional.silu(p).reshape(-1, D))
        new.append(rows[:, n:])
    y = torch.cat(outs)
    out = {"out": y.detach()}
    if carried:
        state[which] = torch.cat(new).detach()
        out["state"] = state
    if train:
        out |= dict(zip(("x_grad", "weight_grad", "bias_grad"), torch.autograd.grad(y, (x, weight, bias), flat["grad"])))
    return out


def _exact_norm(case, s, w):
    names = ["x", "weight"] + (["residual"] if case["residual"] else [])
    x, weight = w["x"], w["weight"].requires_grad_()
    total = x + w["residual"] if case["residual"] else x
    if case["residual"] not in ("", "float32"):  # what is stored is normalised
        total = total.to(_TYPES[case["residual"]]).double()
    total.requires_grad_()
    y = total / torch.sqrt(total.square().mean(-1, keepdim=True) + _EPS) * weight
    out = {"sum": total.detach()} if case["residual"] else {}
    if case["eight"]:
        y, limit = y.detach(), 127.0 if case["eight"] == "int8" else 448.0
        most = y.abs().amax(-1)
        scale = torch.where(most > 0, most / limit, torch.ones_like(most))
        q = y / scale[..., None]
        q = torch.round(q) * scale[..., None] if case["eight"] == "int8" else q.to(_TYPES["float8"]).double()
        return out | {"out": q, "scale": scale}
    onto, dw = torch.autograd.grad(y, (total, weight), w["grad"])
    if case["residual"]:
        onto = onto + w["residual_grad"]
        out["residual_grad"] = onto
    return out | {"out": y.detach(), "x_grad": onto, "weight_grad": dw}
