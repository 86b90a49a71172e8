"""
The operators of a linear attention layer in a language model, as cases that can be timed and compared.

  attend  ``linear_attention`` over whole prompts (``mode`` "prompt"), with its gradients ("train"), and
          ``linear_attention_step`` for one token of each sequence ("step")
  norm    ``group_norm``, the norm of every head's output with its gate or activation, "prompt" and "train"

Fields of a case besides ``op`` and ``mode``: ``dtype`` (of the activations; logs of decays, states and parameters are
float32), ``batch`` and ``T`` (the tokens; a step's ``batch`` is the sequences that take one token), and

  attend  ``heads`` of values, ``groups`` of them that share queries and keys, ``K`` and ``V`` (a head's channels of keys
          and of values), ``decay`` ("token": one for each token and head, "head": one for each head), ``packed``
          (``batch`` sequences of different lengths, some of them empty, behind each other in ``batch * T`` tokens),
          ``state`` (prompts: a state is handed in and the new one handed back)
  norm    ``D`` channels in ``groups``, ``gate`` (z is given), ``act`` ("" or "silu"), ``affine`` (weight and bias)

``own`` is set from outside: false computes the plain form in 32 bits, true calls the framework.
"""
import math

import numpy as np
import torch

own = False

_TYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
_SIZE = {"float32": 4, "bfloat16": 2, "float16": 2}
_EPS = 1e-5
_CHUNK = 64


def _attend(name, mode, dtype, batch, T, heads, K, V, groups=None, decay="token", packed=False, state=False):
    return {"name": name, "op": "attend", "mode": mode, "dtype": dtype, "batch": batch, "T": T, "heads": heads, "groups": groups or heads,
            "K": K, "V": V, "decay": decay, "packed": packed, "state": state}


def _norm(name, mode, dtype, batch, T, D, groups, gate=True, act="", affine=True):
    return {"name": name, "op": "norm", "mode": mode, "dtype": dtype, "batch": batch, "T": T, "D": D, "groups": groups, "gate": gate,
            "act": act, "affine": affine}


def listed():
    return [
        # One token of one user's answer: the call itself is all there is.
        _attend("attend_step_one", "step", "bfloat16", 1, 1, 16, 128, 128),
        # One token of each of many answers that are served together.
        _attend("attend_step_many", "step", "bfloat16", 256, 1, 16, 128, 128),
        # A short prompt in float32, of an odd length, to a small model that decays at a pace of its own in each head.
        _attend("attend_prompt_short", "prompt", "float32", 1, 173, 8, 64, 64, decay="head", state=True),
        # Prompts of different lengths behind each other, as a server takes them in.
        _attend("attend_prompts_packed", "prompt", "bfloat16", 13, 617, 16, 128, 128, packed=True, state=True),
        # One long document: there is more time than there are heads, and their sizes are no whole tiles.
        _attend("attend_long_train", "train", "float32", 1, 30001, 4, 48, 72),
        # A training step whose heads share queries and keys, as the selective scan's channels share B and C.
        _attend("attend_shared_train", "train", "float16", 4, 2048, 32, 128, 64, groups=2),
        # A training step of the large layer at training batch size.
        _attend("attend_layer_train", "train", "bfloat16", 8, 4096, 16, 128, 128),
        # The norm of a served token's heads, gated.
        _norm("norm_token", "prompt", "bfloat16", 16, 1, 2048, 16),
        # ... of a prompt's, where a head is no whole number of vectors.
        _norm("norm_prompt_odd", "prompt", "float16", 8, 2048, 2050, 10, act="silu"),
        # ... of a small model's training step, ungated and in float32.
        _norm("norm_small_train", "train", "float32", 4, 1001, 512, 8, gate=False),
        # ... of the large layer's.
        _norm("norm_layer_train", "train", "bfloat16", 8, 4096, 2048, 16),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi))))))))


# The most products of keys with values (tokens x heads x K x V) and values (tokens x heads x the larger of K and V) of one
# drawn call: the listed layers'. A step's states are read and written: fewer of them.
_MOST_PRODUCTS, _MOST_VALUES, _MOST_STATES = 1 << 33, 1 << 26, 1 << 26


def draw(rng):
    dtype = rng.choices(("float32", "bfloat16", "float16"), (0.3, 0.5, 0.2))[0]
    if rng.random() < 0.35:
        groups = rng.choice((1, 2, 4, 8, 10, 16, 24))
        each = _log_int(rng, 8, 4096 // groups)
        if rng.random() < 0.6:  # the widths that models choose
            each = max(8, each - each % 8)
        D, mode = groups * each, rng.choice(("prompt", "train"))
        rows = _log_int(rng, 1, _MOST_VALUES // D)
        batch = _log_int(rng, 1, min(rows, 64))
        gate = rng.random() < 0.6
        case = _norm("", mode, dtype, batch, max(1, rows // batch), D, groups, gate, rng.choice(("", "" if gate else "silu")), rng.random() < 0.8)
        del case["name"]
        return case
    mode = rng.choices(("step", "prompt", "train"), (0.25, 0.4, 0.35))[0]
    K, V = (rng.choice((32, 64, 64, 128, 128, 256)) if rng.random() < 0.6 else _log_int(rng, 8, 256) for _ in range(2))
    heads = _log_int(rng, 1, max(1, 4096 // max(K, V)))
    most = min(_MOST_VALUES // (heads * max(K, V)), _MOST_PRODUCTS // (heads * K * V))
    if dtype == "float32":
        most //= 2  # (as many bytes as the listed ones)
    if mode == "step":
        batch, T = _log_int(rng, 1, max(1, min(512, _MOST_STATES // (heads * K * V)))), 1
    else:
        tokens = _log_int(rng, 16, min(most, 1 << 17))
        batch = _log_int(rng, 1, min(64, tokens))
        T = min(32768, max(1, tokens // batch))
    groups = rng.choice([heads, heads, heads] + [g for g in (1, 2, 4) if heads % g == 0])
    packed = mode != "step" and batch > 1 and rng.random() < 0.4
    state = mode == "prompt" and rng.random() < 0.6
    case = _attend("", mode, dtype, batch, T, heads, K, V, groups, rng.choice(("token", "token", "head")), packed, state)
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
    dtype, train, step = _TYPES[case["dtype"]], case["mode"] == "train", case["mode"] == "step"
    packed = case.get("packed", False)
    lead = (case["batch"],) if step else (1, case["batch"] * case["T"]) if packed else (case["batch"], case["T"])

    def normal(*shape, of=dtype, scale=1.0, at=0.0):
        return torch.randn(shape, generator=gen, device="cuda").mul_(scale).add_(at).to(of)

    def leaf(t):
        return t.detach().requires_grad_(train)

    s = {"case": case}
    if case["op"] == "norm":
        D = case["D"]
        s["x"] = leaf(normal(*lead, D, scale=2.0, at=0.1))
        s["weight"] = leaf(normal(D, of=torch.float32, scale=0.1, at=1.0)) if case["affine"] else None
        s["bias"] = leaf(normal(D, of=torch.float32, scale=0.1)) if case["affine"] else None
        # (the gate is the second half of the projection that gives the layer's first input as well)
        s["z"] = leaf(normal(*lead, 2 * D)[..., D:]) if case["gate"] else None
        if train:
            s["grad"] = normal(*lead, D)
        return s
    H, G, K, V = (case[n] for n in ("heads", "groups", "K", "V"))
    sequences, slots = case["batch"], case["batch"] + 3  # (steps: more states are kept than take a token)
    # Queries, keys and values are parts of one projection.
    parts = normal(*lead, 2 * G * K + H * V)
    s["q"], s["k"] = (leaf(parts[..., a:a + G * K].unflatten(-1, (G, K))) for a in (0, G * K))
    s["v"] = leaf(parts[..., 2 * G * K:].unflatten(-1, (H, V)))
    # Every head has a pace of its own, from hundreds of tokens to one or two; tokens choose around it.
    pace = torch.rand(H, generator=gen, device="cuda").mul_(math.log(500.0)).add_(math.log(2e-3)).exp_()
    if case["decay"] == "head":
        s["decay"] = leaf(-pace)
    else:
        s["decay"] = leaf(-pace * torch.log1p(torch.exp(normal(*lead, H, of=torch.float32, at=0.5))))
    if packed:
        s["offsets"] = torch.from_numpy(np.concatenate([[0], np.cumsum(_lengths(case, seed))]).astype(np.int32)).cuda()
    if step:
        s["slots"] = torch.randperm(slots, generator=gen, device="cuda")[:sequences].to(torch.int32)
    if step or case["state"]:
        s["state"] = normal(slots if step else sequences, H, K, V, of=torch.float32)
    if train:
        s["grad"] = normal(*lead, H, V)
    return s


def run(s):
    case = s["case"]
    if own:
        return _run_own(case, s)
    with torch.no_grad():
        return (_plain_attend if case["op"] == "attend" else _plain_norm)(case, s)


# ---------------------------------------------------------------------------------------------- the framework's calls
def _run_own(case, s):
    import scanscam_amd as f

    mode = case["mode"]
    if case["op"] == "norm":
        got = f.group_norm(s["x"], case["groups"], s["weight"], s["bias"], s["z"], eps=_EPS, activation=case["act"] or None)
        names = ["x"] + (["weight", "bias"] if case["affine"] else []) + (["z"] if case["gate"] else [])
    else:
        names, scale = ["q", "k", "v", "decay"], case["K"] ** -0.5
        given = [s[n] for n in names]
        if mode == "step":
            out = f.linear_attention_step(s["state"], *given, scale=scale, slots=s["slots"])
            return {"out": out, "state": s["state"]}
        got = f.linear_attention(*given, scale=scale, state=s.get("state"), offsets=s.get("offsets"), return_state=case["state"])
    if mode == "prompt":
        return {"out": got[0], "state": got[1]} if case.get("state") else {"out": got}
    grads = torch.autograd.grad(got, [s[n] for n in names], s["grad"])
    return {"out": got.detach()} | {n + "_grad": g for n, g in zip(names, grads)}


# ------------------------------------------------------------------------------------------------------- plain forms
def _doubled(a, b):
    """h[c] = a[c] h[c-1] + b[c] along the first dimension; a is a number for each of b's leading two."""
    span = 1
    while span < a.shape[0]:
        b = torch.cat((b[:span], torch.addcmul(b[span:], a[span:, :, None, None], b[:-span])))
        a = torch.cat((a[:span], a[span:] * a[:-span]))
        span *= 2
    return b


def _chunks(case, s):
    """Chunks of 64 tokens that never cross a sequence's border: the token of each place (one past the last where there is
    none), its sequence, and whether a chunk is the first or the last of its sequence."""
    S, M = case["batch"], case["batch"] * case["T"]
    ends = s["offsets"].long() if "offsets" in s else torch.arange(S + 1, device="cuda") * case["T"]
    begin, length = ends[:-1], ends[1:] - ends[:-1]
    upto = ((length + _CHUNK - 1) // _CHUNK).cumsum(0)
    c = torch.arange(M // _CHUNK + S, device="cuda")
    of = torch.bucketize(c, upto, right=True).clamp_(max=S - 1)
    number = c - torch.cat((upto.new_zeros(1), upto[:-1]))[of]
    place = number[:, None] * _CHUNK + torch.arange(_CHUNK, device="cuda")
    there = place < length[of, None]
    token = torch.where(there, begin[of, None] + place, M)
    return token, of, (number == 0) & there[:, 0], ((number + 1) * _CHUNK >= length[of]) & there[:, 0]


def _plain_attend(case, s):
    H, G, K, V, dtype = case["heads"], case["groups"], case["K"], case["V"], _TYPES[case["dtype"]]
    scale, M = K ** -0.5, case["batch"] * case["T"]
    if case["mode"] == "step":
        q, k = (s[n].float().repeat_interleave(H // G, 1) for n in "qk")
        slots = s["slots"].long()
        h = torch.exp(s["decay"].expand(M, H))[..., None, None] * s["state"][slots] + k.unsqueeze(-1) * s["v"].float().unsqueeze(-2)
        s["state"][slots] = h
        return {"out": ((q * scale).unsqueeze(-1) * h).sum(-2).to(dtype), "state": s["state"]}
    token, of, first, last = _chunks(case, s)

    def chunked(t):  # [chunks, heads, 64, ...], zeros where there is no token
        t = torch.cat((t, torch.zeros_like(t[:1])))[token]
        return t.transpose(1, 2)

    def back(t, name, sizes):  # the tokens' own, in their order
        out = t.new_empty(M + 1, *sizes)
        out[token.reshape(-1)] = t.transpose(1, 2).reshape(-1, *sizes)
        return out[:M].view(s[name].shape[:2] + sizes)

    q, k = (chunked(s[n].float().reshape(M, G, K).repeat_interleave(H // G, 1)) for n in "qk")
    v = chunked(s["v"].float().reshape(M, H, V))
    q = q * scale
    logs = (s["decay"].expand(M, H) if s["decay"].dim() == 1 else s["decay"].reshape(M, H)).double()
    sums = chunked(logs).cumsum(-1)  # (in 64 bits: differences of long sums)
    end = sums[..., -1:]
    before = sums.unsqueeze(-1) - sums.unsqueeze(-2)
    lower = torch.ones(_CHUNK, _CHUNK, dtype=torch.bool, device="cuda").tril()
    weight = torch.where(lower, before, -math.inf).float().exp()
    del before
    into, onto, whole = sums.float().exp().unsqueeze(-1), (end - sums).float().exp().unsqueeze(-1), end.squeeze(-1).float().exp()
    local = (k * onto).transpose(-1, -2) @ v
    keep = torch.where(first[:, None], 0.0, whole)
    kept = {}
    if case["state"]:
        start = s["state"][of]
        local = local + torch.where(first[:, None, None, None], whole[..., None, None] * start, 0.0)
    after = _doubled(keep, local)
    del local
    ahead = torch.cat((torch.zeros_like(after[:1]), after[:-1]))
    ahead = torch.where(first[:, None, None, None], start if case["state"] else 0.0, ahead)
    if case["state"]:
        new = s["state"].clone()
        new[of[last]] = after[last]
        kept["state"] = new
    del after
    scores = q @ k.transpose(-1, -2)
    out = (q * into) @ ahead + (scores * weight) @ v
    kept["out"] = back(out, "v", (H, V)).to(dtype)
    if case["mode"] != "train":
        return kept
    g = chunked(s["grad"].float().reshape(M, H, V))
    values = g @ v.transpose(-1, -2)
    local = (q * into).transpose(-1, -2) @ g
    later = _doubled(torch.where(last[:, None], 0.0, whole).flip(0), local.flip(0)).flip(0)
    del local
    later = torch.cat((later[1:], torch.zeros_like(later[:1])))
    later = torch.where(last[:, None, None, None], 0.0, later)
    dq = (g * into) @ ahead.transpose(-1, -2)
    dk = (v * onto) @ later.transpose(-1, -2)
    # A decay's gradient is what passes it: from states to tokens, from tokens to states, past the whole chunk, inside of it.
    passes = (scores * values * weight).tril(-1)
    inside = (passes.sum(-1) - passes.sum(-2)).double()
    through = whole * (later * ahead).sum((-1, -2))
    reads, writes = (q * dq).sum(-1).double(), (k * dk).sum(-1).double()
    decay = through.unsqueeze(-1) + (reads + inside).flip(-1).cumsum(-1).flip(-1) + writes.cumsum(-1) - writes
    del passes
    dq = (dq + (values * weight) @ k) * scale
    dk = dk + (values * weight).transpose(-1, -2) @ q
    dv = (k * onto) @ later + (scores * weight).transpose(-1, -2) @ g
    kept["v_grad"] = back(dv, "v", (H, V)).to(dtype)
    for name, t in (("q", dq), ("k", dk)):
        t = back(t, name, (H, K))
        kept[name + "_grad"] = t.unflatten(2, (G, H // G)).sum(3).to(dtype)
    decay = back(decay.unsqueeze(-1), "v", (H, 1)).squeeze(-1)
    kept["decay_grad"] = (decay.sum((0, 1)) if case["decay"] == "head" else decay).float()
    return kept


def _plain_norm(case, s):
    G, dtype, shape = case["groups"], _TYPES[case["dtype"]], s["x"].shape
    split = lambda t: t.unflatten(-1, (G, -1))  # noqa: E731
    x = split(s["x"].float())
    x = x - x.mean(-1, keepdim=True)
    rstd = torch.rsqrt((x * x).mean(-1, keepdim=True) + _EPS)
    unit = x * rstd
    u = unit if not case["affine"] else unit * split(s["weight"]) + split(s["bias"])
    sig = lambda t: 1.0 / (1.0 + torch.exp(-t))  # noqa: E731
    a = u * sig(u) if case["act"] else u
    y = a
    if case["gate"]:
        z = split(s["z"].float())
        y = a * (z * sig(z))
    kept = {"out": y.reshape(shape).to(dtype)}
    if case["mode"] != "train":
        return kept
    g = split(s["grad"].float())
    if case["gate"]:
        kept["z_grad"] = (g * a * sig(z) * (1.0 + z * (1.0 - sig(z)))).reshape(shape).to(dtype)
        g = g * (z * sig(z))
    if case["act"]:
        g = g * sig(u) * (1.0 + u * (1.0 - sig(u)))
    if case["affine"]:
        kept["weight_grad"] = (g * unit).flatten(-2).flatten(0, -2).double().sum(0).float()
        kept["bias_grad"] = g.flatten(-2).flatten(0, -2).double().sum(0).float()
        g = g * split(s["weight"])
    g = rstd * (g - g.mean(-1, keepdim=True) - unit * (g * unit).mean(-1, keepdim=True))
    kept["x_grad"] = g.reshape(shape).to(dtype)
    return kept


# ------------------------------------------------------------------------------------------------------------- cost
def work(case):
    size, M = _SIZE[case["dtype"]], case["batch"] * case["T"]
    train = case["mode"] == "train"
    if case["op"] == "norm":
        D, params = case["D"], 8 * case["D"] if case["affine"] else 0
        gate, act = (1 if case["gate"] else 0), (1 if case["act"] else 0)
        if train:  # x, z -> y; x, z, y's grad -> the grads of x, z
            return {"bytes": M * D * size * (4 + 2 * gate) + 2 * params, "flops": M * D * (24 + 14 * gate + 14 * act)}
        return {"bytes": M * D * size * (2 + gate) + params, "flops": M * D * (8 + 5 * gate + 5 * act)}
    H, G, K, V = (case[n] for n in ("heads", "groups", "K", "V"))
    decays = 4 * H * (M if case["decay"] == "token" else 1)
    kept = 2 * case["batch"] * H * K * V * 4 if case["mode"] == "step" or case["state"] else 0
    keys, values = M * G * K * size, M * H * V * size
    flops = M * H * K * V * 5  # the decay's product, what is written, what is read
    if train:  # q, k, v -> out; q, k, v, out's grad -> the grads of the first three
        return {"bytes": 4 * keys + 4 * values + 2 * decays, "flops": flops + M * H * K * V * 12}
    return {"bytes": 2 * keys + 2 * values + decays + kept, "flops": flops}


# -------------------------------------------------------------------------------------------- the definition in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    w = {n: t.detach().double() for n, t in s.items() if isinstance(t, torch.Tensor) and t.is_floating_point()}
    if case["op"] == "norm":
        return _exact_norm(case, s, w)
    batch, H, G, K, V = (case[n] for n in ("batch", "heads", "groups", "K", "V"))
    M, step, train = batch * case["T"], case["mode"] == "step", case["mode"] == "train"
    if step:
        starts, counts, rows = list(range(batch)), [1] * batch, s["slots"].long()
    else:
        counts = _lengths(case, seed).tolist() if case["packed"] else [case["T"]] * batch
        starts, rows = (np.cumsum(counts) - counts).tolist(), torch.arange(batch, device="cuda")
    # Sequences side by side, the longest first, so that one step serves all that have a token there.
    order = sorted(range(batch), key=lambda i: -counts[i])
    at = torch.tensor([starts[i] for i in order], device="cuda")
    rows = rows[torch.tensor(order, device="cuda")]
    longest = counts[order[0]]
    if longest * (2 if train else 1) * max(60e-6, 4 * batch * H * K * V * 8 / 2e12) > 15.0:
        return None
    lives = np.searchsorted(-np.array([counts[i] for i in order]), -np.arange(longest), side="left").tolist()
    of = torch.arange(H, device="cuda") // (H // G)
    q, k = (w[n].reshape(M, G, K) for n in "qk")
    q = q * K ** -0.5
    v = w["v"].reshape(M, H, V)
    gates = torch.exp(w["decay"]).expand(M, H) if case["decay"] == "head" else torch.exp(w["decay"].reshape(M, H))
    carried = step or case["state"]
    h = w["state"][rows].clone() if carried else torch.zeros(batch, H, K, V, dtype=torch.float64, device="cuda")
    out = torch.empty(M, H, V, dtype=torch.float64, device="cuda")
    g = w["grad"].reshape(M, H, V) if train else None
    dq = torch.empty(M, H, K, dtype=torch.float64, device="cuda") if train else None
    for t in range(longest):
        n = lives[t]
        i, now = at[:n] + t, h[:n]
        now.mul_(gates[i][..., None, None]).addcmul_(k[i][:, of].unsqueeze(-1), v[i].unsqueeze(-2))
        out[i] = (q[i][:, of].unsqueeze(-1) * now).sum(-2)
        if train:
            dq[i] = (now * g[i].unsqueeze(-2)).sum(-1)
    got = {"out": out.reshape(s["v"].shape)}
    if carried:
        state = w["state"].clone()
        state[rows] = h
        got["state"] = state
    if not train:
        return got
    h.zero_()
    dk, dv = torch.empty_like(dq), torch.empty_like(v)
    for t in range(longest - 1, -1, -1):
        n = lives[t]
        i, now = at[:n] + t, h[:n]
        now.addcmul_(q[i][:, of].unsqueeze(-1), g[i].unsqueeze(-2))
        dk[i] = (now * v[i].unsqueeze(-2)).sum(-1)
        dv[i] = (now * k[i][:, of].unsqueeze(-1)).sum(-2)
        now.mul_(gates[i][..., None, None])
    # What a token reads less what it writes, summed up from the end of its sequence.
    passing = (q[:, of] * dq).sum(-1) - (k[:, of] * dk).sum(-1)
    decay = torch.empty_like(passing)
    for b, n in zip(starts, counts):
        decay[b:b + n] = passing[b:b + n].flip(0).cumsum(0).flip(0)
    got["q_grad"] = (dq * K ** -0.5).view(M, G, H // G, K).sum(2).reshape(s["q"].shape)
    got["k_grad"] = dk.view(M, G, H // G, K).sum(2).reshape(s["k"].shape)
    got["v_grad"] = dv.reshape(s["v"].shape)
    got["decay_grad"] = decay.sum(0) if case["decay"] == "head" else decay.reshape(s["decay"].shape)
    return got


def _exact_norm(case, s, w):
    names = [n for n in ("x", "weight", "bias", "z") if n in w]
    train = case["mode"] == "train"
    for n in names:
        w[n].requires_grad_(train)
    x = w["x"].reshape(*s["x"].shape[:-1], case["groups"], -1)
    unit = ((x - x.mean(-1, keepdim=True)) / torch.sqrt(x.var(-1, unbiased=False, keepdim=True) + _EPS)).reshape(s["x"].shape)
    y = unit * w["weight"] + w["bias"] if case["affine"] else unit
    if case["act"]:
        y = torch.nn.functional.silu(y)
    if case["gate"]:
        y = y * torch.nn.functional.silu(w["z"])
    got = {"out": y.detach()}
    if train:
        got |= {n + "_grad": t for n, t in zip(names, torch.autograd.grad(y, [w[n] for n in names], w["grad"]))}
    return got
