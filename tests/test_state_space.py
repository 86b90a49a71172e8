"""
The state space layer's operators without a GPU: the plain loops that CPU tensors take (and that the kernels are tested
against), what the entry points refuse, and the C ABI's checks of arguments. No kernel is launched in this file.
"""
import ctypes
import os
import re
import subprocess

import pytest
import torch

import scanscam_amd as f
from scanscam_amd import baseline, hip, state_space

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HEADER = os.path.join(ROOT, "include", "scanscam_ops.h")
E_OK, E_INVAL, E_DTYPE, E_ALIGN, E_PLAN, E_WORKSPACE, E_LAUNCH = range(7)


def inputs(batch=2, T=5, D=6, N=3, groups=1, dtype=torch.float32, seed=0):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(s, generator=g)  # noqa: E731
    v = dict(x=r(batch, T, D), dt=r(batch, T, D), A=-r(D, N).exp(), B=r(batch, T, groups, N), C=r(batch, T, groups, N), D=r(D), z=r(batch, T, D), dt_bias=r(D))
    return {k: t if k in ("A", "D", "dt_bias") else t.to(dtype) for k, t in v.items()}


def test_plain_scan_is_the_framework_s_scan():
    """With A, B and C written out, the recurrence is scan()'s: h[t] = exp(d A) h[t-1] + d x B."""
    v = inputs(groups=2)
    d = torch.nn.functional.softplus(v["dt"] + v["dt_bias"])
    B, C = (v[k].repeat_interleave(3, 2) for k in "BC")
    gate, value = torch.exp(d[..., None] * v["A"]), (d * v["x"])[..., None] * B
    h = f.scan(gate.movedim(1, -1), value.movedim(1, -1)).movedim(-1, 1)
    want = ((C * h).sum(-1) + v["D"] * v["x"]) * torch.nn.functional.silu(v["z"])
    y, state = f.selective_scan(**v, softplus=True, return_state=True)
    torch.testing.assert_close(y, want, rtol=1e-5, atol=1e-6)
    torch.testing.assert_close(state, h[:, -1], rtol=1e-5, atol=1e-6)


def test_plain_forms_have_the_gradients_of_differences():
    g = torch.Generator().manual_seed(1)
    wide = {k: t.double().requires_grad_() for k, t in inputs(1, 4, 2, 2).items()}
    state = torch.randn(1, 2, 2, generator=g, dtype=torch.float64, requires_grad=True)
    names = list(wide)
    torch.autograd.gradcheck(lambda s, *t: baseline.naive_selective_scan(**dict(zip(names, t)), softplus=True, state=s, return_state=True), (state, *wide.values()))
    x, w, b, s = (torch.randn(n, generator=g, dtype=torch.float64, requires_grad=True) for n in ((2, 3, 2), (2, 3), (2,), (2, 2, 2)))
    torch.autograd.gradcheck(lambda x, w, b, s: baseline.naive_causal_conv(x, w, b, activation="silu", state=s, return_state=True), (x, w, b, s))
    r, v = (torch.randn(n, generator=g, dtype=torch.float64, requires_grad=True) for n in ((2, 3, 2), (2,)))
    torch.autograd.gradcheck(lambda x, v, r: baseline.naive_rms_norm(x, v, r), (x, v, r))


def test_packed_sequences_are_sequences_alone():
    v, offsets = inputs(1, 9), torch.tensor([0, 4, 4, 9])
    y, state = f.selective_scan(**v, offsets=offsets, return_state=True)
    seqs = ("x", "dt", "B", "C", "z")
    for s, (a, b) in enumerate([(0, 4), (4, 4), (4, 9)]):
        one, end = f.selective_scan(**{k: t[:, a:b] if k in seqs else t for k, t in v.items()}, return_state=True)
        assert torch.equal(y[:, a:b], one) and torch.equal(state[s], end[0])
    w = torch.randn(6, 4)
    y, state = f.causal_conv(v["x"], w, offsets=offsets, return_state=True)
    for s, (a, b) in enumerate([(0, 4), (4, 4), (4, 9)]):
        one, end = f.causal_conv(v["x"][:, a:b], w, return_state=True)
        assert torch.equal(y[:, a:b], one) and torch.equal(state[s], end[0])


def test_single_tokens_continue_a_prompt():
    v, w = inputs(2, 6), torch.randn(6, 4)
    seqs = ("x", "dt", "B", "C", "z")
    want, end = f.selective_scan(**v, softplus=True, return_state=True)
    _, state = f.selective_scan(**{k: t[:, :5] if k in seqs else t for k, t in v.items()}, softplus=True, return_state=True)
    last = {k: t[:, 5] if k in seqs else t for k, t in v.items()}
    y = f.selective_scan_step(state, **last, softplus=True)
    torch.testing.assert_close(y, want[:, 5])
    torch.testing.assert_close(state, end)
    want, end = f.causal_conv(v["x"], w, activation="silu", return_state=True)
    _, state = f.causal_conv(v["x"][:, :5], w, activation="silu", return_state=True)
    torch.testing.assert_close(f.causal_conv_step(state, v["x"][:, 5], w, activation="silu"), want[:, 5])
    assert torch.equal(state, end)
    kept = torch.randn(5, 3, 6)
    before = kept.clone()
    y = f.causal_conv_step(kept, v["x"][:, 0], w, slots=torch.tensor([-1, 3]))
    assert torch.equal(y[0], torch.zeros(6)) and torch.equal(kept[[0, 1, 2, 4]], before[[0, 1, 2, 4]]) and not torch.equal(kept[3], before[3])


@pytest.mark.parametrize("quant,limit", [(torch.int8, 127), (torch.float8_e4m3fn, 448)])
def test_norm_in_eight_bits(quant, limit):
    x = torch.randn(4, 10)
    x[2] = 0
    q, scale, total = f.rms_norm(x, torch.ones(10), x * 2, quant=quant)
    assert q.dtype == quant and scale.shape == (4,) and torch.equal(total, x + x * 2)
    assert float(scale[2]) == 1.0 and q.float().abs().amax(-1).tolist() == [limit, limit, 0, limit]


def test_what_the_scan_refuses():
    v = inputs()
    bad = lambda **k: f.selective_scan(**{**v, **k})  # noqa: E731
    for case in ({"x": v["x"][0]}, {"dt": v["dt"][:, :4]}, {"A": v["A"][:5]}, {"A": torch.zeros(6, 257)}, {"C": v["C"][..., :2]}, {"D": v["D"][:3]},
                 {"z": v["z"][:1]}, {"dt_bias": v["A"]}, {"state": torch.zeros(3, 6, 3)}, {"B": torch.zeros(2, 5, 4, 3), "C": torch.zeros(2, 5, 4, 3)},
                 {"offsets": torch.tensor([0, 5])}, {"B": torch.zeros(2, 5)}):
        with pytest.raises(AssertionError, match="selective_scan"):
            bad(**case)
    for case in ({"x": v["x"].double()}, {"dt": v["dt"].half()}, {"A": v["A"].double()}, {"state": torch.zeros(2, 6, 3, dtype=torch.bfloat16)}):
        with pytest.raises(TypeError, match="selective_scan"):
            bad(**case)
    one = {k: t[:1] if t.dim() > 2 else t for k, t in v.items()}
    with pytest.raises(TypeError, match="offsets"):
        f.selective_scan(**one, offsets=torch.tensor([0.0, 5.0]))
    with pytest.raises(AssertionError, match="offsets"):
        f.selective_scan(**one, offsets=torch.tensor([5]))
    with pytest.raises(RuntimeError, match="meta"):
        bad(D=torch.empty(6, device="meta"))


def test_what_the_step_refuses():
    v, state = {k: t[:, 0] if t.dim() > 2 else t for k, t in inputs().items()}, torch.zeros(4, 6, 3)
    slots = torch.tensor([1, 0])
    for error, case in ((AssertionError, {}), (AssertionError, {"slots": slots[:1]}), (TypeError, {"slots": slots.float()}), (AssertionError, {"dt": v["dt"][:, :2], "slots": slots}),
                        (AssertionError, {"state": state[..., :2], "slots": slots}), (RuntimeError, {"state": torch.zeros(4, 3, 6).mT, "slots": slots}),
                        (TypeError, {"state": state.half(), "slots": slots}), (RuntimeError, {"x": v["x"].clone().requires_grad_(), "slots": slots}),
                        (RuntimeError, {"state": state.clone().requires_grad_(), "slots": slots})):
        with pytest.raises(error, match="selective_scan_step"):
            f.selective_scan_step(**{"state": state, **v, **case})
    x, w, kept = torch.zeros(2, 6), torch.zeros(6, 4), torch.zeros(2, 3, 6)
    for error, case in ((AssertionError, {"weight": torch.zeros(6, 9)}), (ValueError, {"activation": "gelu"}), (AssertionError, {"state": kept[:, :2]}),
                        (TypeError, {"state": kept.half()}), (AssertionError, {"bias": torch.zeros(5)}), (RuntimeError, {"weight": w.clone().requires_grad_()})):
        with pytest.raises(error, match="causal_conv_step"):
            f.causal_conv_step(**{"state": kept, "x": x, "weight": w, **case})


def test_what_the_convolution_and_the_norm_refuse():
    x, w = torch.zeros(2, 5, 6), torch.zeros(6, 4)
    for error, case in ((AssertionError, {"x": x[0]}), (AssertionError, {"weight": w[:5]}), (AssertionError, {"weight": torch.zeros(6, 0)}), (ValueError, {"activation": "relu"}),
                        (AssertionError, {"bias": torch.zeros(1)}), (AssertionError, {"state": torch.zeros(2, 4, 6)}), (TypeError, {"state": torch.zeros(2, 3, 6).half()}),
                        (TypeError, {"x": x.double()}), (AssertionError, {"offsets": torch.tensor([0, 5])})):
        with pytest.raises(error, match="causal_conv"):
            f.causal_conv(**{"x": x, "weight": w, **case})
    v = torch.ones(6)
    for error, case in ((AssertionError, {"weight": v[:5]}), (AssertionError, {"residual": x[:1]}), (TypeError, {"quant": torch.uint8}), (TypeError, {"x": x.double()}),
                        (TypeError, {"residual": x.double()}), (RuntimeError, {"x": x.clone().requires_grad_(), "quant": torch.int8}),
                        (AssertionError, {"x": torch.zeros(1, 32769), "weight": torch.zeros(32769)})):
        with pytest.raises(error, match="rms_norm"):
            f.rms_norm(**{"x": x, "weight": v, **case})


def test_header_is_plain_c_and_every_symbol_is_exported(tmp_path):
    src = tmp_path / "t.c"
    structs = ("selective", "selective_step", "conv", "conv_step", "norm")
    src.write_text('#include <stdio.h>\n#include "scanscam_ops.h"\nint main(void) { ' +
                   "".join(f'printf("%zu ", sizeof(scanscam_{s}));' for s in structs) + "return 0; }\n")
    subprocess.run(["gcc", "-std=c99", "-Wall", "-Werror", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(tmp_path / "t")], check=True)
    sizes = [int(n) for n in subprocess.run([str(tmp_path / "t")], check=True, capture_output=True, text=True).stdout.split()]
    mine = (state_space._Selective, state_space._SelectiveStep, state_space._Conv, state_space._ConvStep, state_space._Norm)
    assert sizes == [ctypes.sizeof(s) for s in mine]
    text = re.sub(r"/\*.*?\*/", "", open(HEADER).read(), flags=re.S)
    names = set(re.findall(r"\b(scanscam_[a-z_]+)\s*\(", text))
    assert len(names) == 12
    raw = ctypes.CDLL(hip.LIB_PATH)
    for name in names:
        assert hasattr(raw, name), name


def test_the_library_checks_its_arguments_before_any_launch():
    L, fake = state_space._lib(), 0x10000  # never dereferenced: every call below must fail first
    T, P = state_space._Tokens, state_space._Param

    def scan(**k):
        a = state_space._Selective(batch=1, T=4, sequences=1, channels=8, groups=1, N=4, dtype=0)
        for n in ("x", "dt", "B", "C", "y", "gy", "gx", "gdt", "gB", "gC"):
            setattr(a, n, T(fake, 64, 8, 4))
        a.A, a.gA, a.saved = P(fake, 0), fake, fake
        for n, v in k.items():
            setattr(a, n, v)
        return a

    for rc, k in ((E_INVAL, {"N": 0}), (E_INVAL, {"N": 257}), (E_INVAL, {"groups": 3}), (E_INVAL, {"T": -1}), (E_INVAL, {"sequences": 2}), (E_DTYPE, {"dtype": 3}),
                  (E_INVAL, {"x": T(None, 1, 1, 1)}), (E_INVAL, {"x": T(fake, -1, 1, 1)}), (E_ALIGN, {"x": T(fake + 2, 1, 1, 1)}), (E_INVAL, {"A": P(None, 0)}),
                  (E_DTYPE, {"A": P(fake, 3)}), (E_ALIGN, {"A": P(fake + 2, 0)}), (E_INVAL, {"offsets": fake, "batch": 2}), (E_ALIGN, {"offsets": fake + 4, "offsets64": 1}),
                  (E_INVAL, {"y": T(None, 1, 1, 1)}), (E_ALIGN, {"state_in": fake + 2}), (E_INVAL, {"channels": 1 << 21})):
        assert L.scanscam_selective_fwd(scan(**k), None) == rc, k
    assert L.scanscam_selective_bwd(scan(), None) == E_WORKSPACE
    assert L.scanscam_selective_bwd(scan(saved=None), None) == E_INVAL
    assert L.scanscam_selective_bwd(scan(gx=T(None, 1, 1, 1)), None) == E_INVAL
    assert L.scanscam_selective_bwd(scan(gA=None), None) == E_INVAL
    assert L.scanscam_selective_workspace_bytes(scan(), hip.BACKWARD) > 0 and L.scanscam_selective_saved_bytes(scan()) > 0
    assert L.scanscam_selective_fwd(scan(sequences=0, batch=0), None) == E_OK and L.scanscam_selective_fwd(scan(channels=0), None) == E_OK

    step = state_space._SelectiveStep(rows=2, channels=8, groups=1, N=4, slots=2, dtype=0)
    assert L.scanscam_selective_step_fwd(step, None) == E_INVAL
    for n in ("x", "dt", "B", "C", "y"):
        setattr(step, n, T(fake, 0, 8, 4))
    step.A = P(fake, 0)
    assert L.scanscam_selective_step_fwd(step, None) == E_INVAL  # no state
    step.state = fake + 1
    assert L.scanscam_selective_step_fwd(step, None) == E_ALIGN

    def conv(**k):
        a = state_space._Conv(batch=1, T=4, sequences=1, channels=8, K=4, dtype=1, x=T(fake, 64, 8, 0), y=T(fake, 64, 8, 0), weight=P(fake, 0), gweight=fake,
                              gy=T(fake, 64, 8, 0), gx=T(fake, 64, 8, 0))
        for n, v in k.items():
            setattr(a, n, v)
        return a

    for rc, k in ((E_INVAL, {"K": 0}), (E_INVAL, {"K": 9}), (E_INVAL, {"activation": 2}), (E_DTYPE, {"dtype": 3}), (E_INVAL, {"x": T(None, 0, 0, 0)}),
                  (E_ALIGN, {"y": T(fake + 1, 0, 0, 0)}), (E_INVAL, {"weight": P(None, 0)}), (E_INVAL, {"sequences": 3}), (E_INVAL, {"batch": 1 << 29, "sequences": 1 << 29})):
        assert L.scanscam_conv_fwd(conv(**k), None) == rc, k
    assert L.scanscam_conv_bwd(conv(), None) == E_WORKSPACE
    assert L.scanscam_conv_bwd(conv(gweight=None), None) == E_INVAL
    assert L.scanscam_conv_step_fwd(state_space._ConvStep(rows=1, channels=8, K=4, dtype=0, x=T(fake, 0, 8, 0), y=T(fake, 0, 8, 0), weight=P(fake, 0)), None) == E_INVAL

    def norm(**k):
        a = state_space._Norm(rows=4, channels=8, x=fake, x_stride=8, weight=P(fake, 0), y=fake, dtype=1, out_dtype=1)
        for n, v in k.items():
            setattr(a, n, v)
        return a

    for rc, k in ((E_INVAL, {"rows": -1}), (E_INVAL, {"channels": 32769}), (E_DTYPE, {"dtype": 9}), (E_DTYPE, {"out_dtype": 0}), (E_INVAL, {"residual": fake}),
                  (E_INVAL, {"x": None}), (E_INVAL, {"y": None}), (E_INVAL, {"out_dtype": 17}), (E_ALIGN, {"x": fake + 1}), (E_INVAL, {"weight": P(None, 0)})):
        assert L.scanscam_norm_fwd(norm(**k), None) == rc, k
    assert L.scanscam_norm_bwd(norm(gweight=fake, gy=fake, gx=fake, rstd=fake), None) == E_WORKSPACE
    assert L.scanscam_norm_bwd(norm(gy=fake, gx=fake, rstd=fake), None) == E_INVAL
