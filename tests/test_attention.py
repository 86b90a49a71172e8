"""
The linear attention layer's operators without a GPU: the plain loops that CPU tensors take (and that the kernels are tested against), what the
entry points refuse, and the C ABI's checks of arguments. No kernel is launched in this file.
"""
import ctypes
import os
import re
import subprocess

import pytest
import torch

import scanscam_amd as f
from scanscam_amd import attention, baseline, hip, state_space

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HEADER = os.path.join(ROOT, "include", "scanscam_attention.h")
E_OK, E_INVAL, E_DTYPE, E_ALIGN, E_PLAN, E_WORKSPACE, E_LAUNCH = range(7)


def inputs(batch=2, T=5, heads=4, groups=2, K=3, V=6, dtype=torch.float32, seed=0):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(s, generator=g)  # noqa: E731
    return dict(q=r(batch, T, groups, K).to(dtype), k=r(batch, T, groups, K).to(dtype), v=r(batch, T, heads, V).to(dtype), decay=-r(batch, T, heads).abs())


def test_plain_attention_is_a_sum_over_the_tokens_before():
    v = {n: t.double() for n, t in inputs().items()}
    q, k = (v[n].repeat_interleave(2, 2) for n in "qk")
    sums = v["decay"].cumsum(1)
    w = (sums[:, :, None] - sums[:, None]).exp() * torch.ones(5, 5).tril()[None, :, :, None]
    want = torch.einsum("bthk,bshk,btsh,bshv->bthv", q, k, w, v["v"]) * 0.3
    torch.testing.assert_close(baseline.naive_linear_attention(**v, scale=0.3), want)


def test_plain_attention_is_the_framework_s_scan():
    """Every value of a state is a scan of its own: S[t] = exp(decay) S[t-1] + k v."""
    v = inputs(groups=4)
    gate = v["decay"].exp()[..., None, None].expand(2, 5, 4, 3, 6)
    value = v["k"].unsqueeze(-1) * v["v"].unsqueeze(-2)
    h = f.scan(gate.movedim(1, -1).contiguous(), value.movedim(1, -1).contiguous()).movedim(-1, 1)
    y, state = f.linear_attention(**v, return_state=True)
    torch.testing.assert_close(y, (v["q"].unsqueeze(-1) * h).sum(-2), rtol=1e-5, atol=1e-6)
    torch.testing.assert_close(state, h[:, -1], rtol=1e-5, atol=1e-6)


def test_plain_forms_have_the_gradients_of_differences():
    wide = {n: t.double().requires_grad_() for n, t in inputs(1, 4, 2, 1, 2, 2).items()}
    g = torch.Generator().manual_seed(1)
    r = lambda *s: torch.randn(s, generator=g, dtype=torch.float64).requires_grad_()  # noqa: E731
    torch.autograd.gradcheck(lambda s, *t: baseline.naive_linear_attention(*t, scale=0.5, state=s, return_state=True), (r(1, 2, 2, 2), *wide.values()))
    fixed = (-torch.rand(2, generator=g, dtype=torch.float64)).requires_grad_()
    torch.autograd.gradcheck(lambda d: baseline.naive_linear_attention(wide["q"].detach(), wide["k"].detach(), wide["v"].detach(), d), (fixed,))
    for activation in (None, "silu"):
        torch.autograd.gradcheck(lambda x, w, b, z: baseline.naive_group_norm(x, 2, w, b, z, activation=activation), (r(3, 6), r(6), r(6), r(3, 6)))


def test_plain_group_norm_is_torch_s():
    x, w, b = torch.randn(7, 12), torch.randn(12), torch.randn(12)
    torch.testing.assert_close(f.group_norm(x, 3, w, b), torch.nn.functional.group_norm(x, 3, w, b))
    torch.testing.assert_close(f.group_norm(x, 1, w, None, activation="silu"), torch.nn.functional.silu(torch.nn.functional.layer_norm(x, (12,), w)))


def test_packed_sequences_are_sequences_alone():
    v, offsets = inputs(1, 9), torch.tensor([0, 4, 4, 9])
    y, state = f.linear_attention(**v, offsets=offsets, return_state=True)
    for s, (a, b) in enumerate([(0, 4), (4, 4), (4, 9)]):
        one, end = f.linear_attention(**{n: t[:, a:b] for n, t in v.items()}, return_state=True)
        assert torch.equal(y[:, a:b], one) and torch.equal(state[s], end[0])


def test_single_tokens_continue_a_prompt():
    v = inputs(2, 6)
    want, end = f.linear_attention(**v, scale=0.5, return_state=True)
    _, state = f.linear_attention(**{n: t[:, :5] for n, t in v.items()}, scale=0.5, return_state=True)
    y = f.linear_attention_step(state, **{n: t[:, 5] for n, t in v.items()}, scale=0.5)
    torch.testing.assert_close(y, want[:, 5])
    torch.testing.assert_close(state, end)
    kept = torch.randn(5, 4, 3, 6)
    before = kept.clone()
    y = f.linear_attention_step(kept, **{n: t[:, 0] for n, t in v.items()}, slots=torch.tensor([-1, 3]))
    assert torch.equal(y[0], torch.zeros(4, 6)) and torch.equal(kept[[0, 1, 2, 4]], before[[0, 1, 2, 4]]) and not torch.equal(kept[3], before[3])


def test_what_attention_refuses():
    v = inputs()
    bad = lambda **k: f.linear_attention(**{**v, **k})  # noqa: E731
    for case in ({"q": v["q"][0]}, {"k": v["k"][:, :4]}, {"k": v["k"][..., :2]}, {"v": v["v"][..., 0]}, {"q": torch.zeros(2, 5, 3, 3), "k": torch.zeros(2, 5, 3, 3)},
                 {"q": torch.zeros(2, 5, 2, 257), "k": torch.zeros(2, 5, 2, 257)}, {"v": torch.zeros(2, 5, 4, 257)}, {"q": torch.zeros(2, 5, 2, 0), "k": torch.zeros(2, 5, 2, 0)},
                 {"q": torch.zeros(1, 5, 2, 3), "k": torch.zeros(1, 5, 2, 3)}, {"decay": v["decay"][:, :4]}, {"decay": torch.zeros(2)}, {"decay": torch.zeros(5, 4)},
                 {"state": torch.zeros(2, 4, 6, 3)}, {"state": torch.zeros(1, 4, 3, 6)}, {"offsets": torch.tensor([0, 5])}, {"q": torch.zeros(2, 5, 0, 3), "k": torch.zeros(2, 5, 0, 3)}):
        with pytest.raises(AssertionError, match="linear_attention"):
            bad(**case)
    for case in ({"v": v["v"].double()}, {"q": v["q"].half()}, {"decay": v["decay"].double()}, {"state": torch.zeros(2, 4, 3, 6, dtype=torch.bfloat16)}):
        with pytest.raises(TypeError, match="linear_attention"):
            bad(**case)
    one = {n: t[:1] for n, t in v.items()}
    with pytest.raises(TypeError, match="offsets"):
        f.linear_attention(**one, offsets=torch.tensor([0.0, 5.0]))
    with pytest.raises(AssertionError, match="offsets"):
        f.linear_attention(**one, offsets=torch.tensor([5]))
    with pytest.raises(RuntimeError, match="meta"):
        bad(decay=torch.empty(4, device="meta"))


def test_what_the_step_refuses():
    v, state, slots = {n: t[:, 0] for n, t in inputs().items()}, torch.zeros(4, 4, 3, 6), torch.tensor([1, 0])
    for error, case in ((AssertionError, {}), (AssertionError, {"slots": slots[:1]}), (TypeError, {"slots": slots.float()}), (AssertionError, {"k": v["k"][:, :, :2], "slots": slots}),
                        (AssertionError, {"state": state[..., :2], "slots": slots}), (AssertionError, {"state": state[0], "slots": slots}), (RuntimeError, {"state": torch.zeros(4, 4, 6, 3).mT, "slots": slots}),
                        (TypeError, {"state": state.half(), "slots": slots}), (RuntimeError, {"v": v["v"].clone().requires_grad_(), "slots": slots}),
                        (RuntimeError, {"state": state.clone().requires_grad_(), "slots": slots}), (AssertionError, {"decay": v["decay"][:, :3], "slots": slots})):
        with pytest.raises(error, match="linear_attention_step"):
            f.linear_attention_step(**{"state": state, **v, **case})


def test_what_the_group_norm_refuses():
    x, w = torch.zeros(2, 5, 6), torch.ones(6)
    for error, case in ((AssertionError, {"groups": 4}), (AssertionError, {"groups": 0}), (AssertionError, {"groups": -1}), (AssertionError, {"x": torch.zeros(())}), (AssertionError, {"weight": w[:5]}),
                        (AssertionError, {"bias": w[:1]}), (AssertionError, {"z": x[:1]}), (TypeError, {"z": x.half()}), (TypeError, {"x": x.double()}), (TypeError, {"weight": w.double()}),
                        (ValueError, {"activation": "gelu"}), (AssertionError, {"x": torch.zeros(1, 8193), "groups": 1})):
        with pytest.raises(error, match="group_norm"):
            f.group_norm(**{"x": x, "groups": 3, **case})


def test_header_is_plain_c_and_every_symbol_is_exported(tmp_path):
    src = tmp_path / "t.c"
    structs = {"attend": attention._Attend, "attend_step": attention._AttendStep, "group_norm": attention._GroupNorm}
    src.write_text('#include <stdio.h>\n#include "scanscam_attention.h"\nint main(void) { ' +
                   "".join(f'printf("%zu ", sizeof(scanscam_{s}));' for s in structs) + "return 0; }\n")
    subprocess.run(["gcc", "-std=c99", "-Wall", "-Werror", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(tmp_path / "t")], check=True)
    sizes = [int(n) for n in subprocess.run([str(tmp_path / "t")], check=True, capture_output=True, text=True).stdout.split()]
    assert sizes == [ctypes.sizeof(s) for s in structs.values()]
    text = re.sub(r"/\*.*?\*/", "", open(HEADER).read(), flags=re.S)
    names = set(re.findall(r"\b(scanscam_[a-z_]+)\s*\(", text))
    assert len(names) == 8
    raw = ctypes.CDLL(hip.LIB_PATH)
    for name in names:
        assert hasattr(raw, name), name


def test_the_library_checks_its_arguments_before_any_launch():
    L, fake = attention._lib(), 0x10000  # never dereferenced: every call below must fail first
    T, P = state_space._Tokens, state_space._Param

    def attend(**k):
        a = attention._Attend(batch=1, T=4, sequences=1, heads=4, groups=2, K=8, V=8, dtype=0, scale=1.0)
        for n in ("q", "k", "v", "y", "gy", "gq", "gk", "gv"):
            setattr(a, n, T(fake, 64, 8, 4))
        for n, v in k.items():
            setattr(a, n, v)
        return a

    shared = ((E_INVAL, {"K": 0}), (E_INVAL, {"K": 257}), (E_INVAL, {"V": 257}), (E_INVAL, {"groups": 3}), (E_INVAL, {"groups": 0}), (E_INVAL, {"T": -1}), (E_INVAL, {"sequences": 2}),
              (E_DTYPE, {"dtype": 3}), (E_INVAL, {"q": T(None, 1, 1, 1)}), (E_INVAL, {"k": T(fake, -1, 1, 1)}), (E_ALIGN, {"v": T(fake + 2, 1, 1, 1)}),
              (E_INVAL, {"k": T(fake, 1, 1 << 22, 1)}), (E_INVAL, {"offsets": fake, "batch": 2}), (E_ALIGN, {"offsets": fake + 4, "offsets64": 1}),
              (E_DTYPE, {"decay": T(fake, 1, 1, 1), "decay_dtype": 5}), (E_ALIGN, {"decay": T(fake + 1, 1, 1, 1), "decay_dtype": 1}), (E_ALIGN, {"state_in": fake + 2}),
              (E_INVAL, {"heads": 1 << 18, "groups": 1}), (E_INVAL, {"parts": -1}), (E_INVAL, {"T": 1 << 31}))
    for rc, k in shared + ((E_INVAL, {"y": T(None, 1, 1, 1)}), (E_WORKSPACE, {"parts": 3})):
        assert L.scanscam_attend_fwd(attend(**k), None) == rc, k
    for rc, k in shared + ((E_INVAL, {"gq": T(None, 1, 1, 1)}), (E_INVAL, {"gy": T(fake, 1, 1 << 22, 1)}), (E_WORKSPACE, {}), (E_INVAL, {"parts": 3, "workspace": fake, "workspace_bytes": 1 << 40}), (E_INVAL, {"gdecay": fake}), (E_ALIGN, {"gstate_in": fake + 1})):
        assert L.scanscam_attend_bwd(attend(**k), None) == rc, k
    assert L.scanscam_attend_fwd(None, None) == L.scanscam_attend_bwd(None, None) == L.scanscam_attend_step_fwd(None, None) == E_INVAL
    assert L.scanscam_attend_fwd(attend(T=0), None) == L.scanscam_attend_fwd(attend(heads=0), None) == E_OK

    def step(**k):
        a = attention._AttendStep(rows=2, heads=4, groups=2, K=8, V=8, slots=2, dtype=0, scale=1.0, state=fake)
        for n in ("q", "k", "v", "y"):
            setattr(a, n, T(fake, 64, 8, 4))
        for n, v in k.items():
            setattr(a, n, v)
        return a

    for rc, k in ((E_INVAL, {"K": 0}), (E_INVAL, {"V": 300}), (E_INVAL, {"groups": 3}), (E_INVAL, {"rows": -1}), (E_INVAL, {"slots": -1}), (E_DTYPE, {"dtype": 7}), (E_INVAL, {"state": None}),
                  (E_ALIGN, {"state": fake + 2}), (E_ALIGN, {"slot": fake + 2}), (E_INVAL, {"y": T(None, 1, 1, 1)}), (E_ALIGN, {"q": T(fake + 1, 1, 1, 1)})):
        assert L.scanscam_attend_step_fwd(step(**k), None) == rc, k
    assert L.scanscam_attend_step_fwd(step(rows=0), None) == E_OK

    def norm(**k):
        a = attention._GroupNorm(rows=2, channels=8, groups=2, x_stride=8, x=fake, y=fake, dtype=0, eps=1e-5, gy=fake, gx=fake)
        for n, v in k.items():
            setattr(a, n, v)
        return a

    shared = ((E_INVAL, {"groups": 3}), (E_INVAL, {"groups": 0}), (E_INVAL, {"channels": 20000}), (E_INVAL, {"x_stride": -1}), (E_INVAL, {"x": None}), (E_DTYPE, {"dtype": 3}), (E_ALIGN, {"x": fake + 2}),
              (E_ALIGN, {"z": fake + 1}), (E_INVAL, {"activation": 2}), (E_DTYPE, {"weight": P(fake, 9)}), (E_ALIGN, {"bias": P(fake + 2, 0)}), (E_INVAL, {"rows": -1}))
    for rc, k in shared + ((E_INVAL, {"y": None}),):
        assert L.scanscam_group_norm_fwd(norm(**k), None) == rc, k
    for rc, k in shared + ((E_INVAL, {"gy": None}), (E_INVAL, {"gz": fake}), (E_INVAL, {"gweight": fake}), (E_INVAL, {"weight": P(fake, 0)}), (E_WORKSPACE, {"weight": P(fake, 0), "gweight": fake})):
        assert L.scanscam_group_norm_bwd(norm(**k), None) == rc, k
    assert L.scanscam_group_norm_fwd(norm(rows=0), None) == E_OK
