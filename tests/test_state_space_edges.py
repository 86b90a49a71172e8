"""
The state space layer's operators at the edges of their arguments, without a GPU.
"""
import os
import subprocess
import sys
import textwrap

import pytest
import torch
from torch.autograd import forward_ad

from scanscam_amd import baseline, causal_conv_step, rms_norm, selective_scan_step


def test_softplus_has_its_gradient_at_zero():
    """The step size's gradient is sigmoid(dt + dt_bias) times what comes in, 1/2 at zero, where projections that start from zeros are."""
    dt = torch.tensor([[[0.0], [-0.0], [1e-30], [3.0], [-90.0], [90.0], [float("-inf")]]], dtype=torch.float64, requires_grad=True)
    x, one, A = torch.ones_like(dt), torch.ones_like(dt), torch.zeros(1, 1, dtype=torch.float64)
    for T in range(dt.shape[1]):
        # With A = 0, B = C = x = 1 the last token adds its own step size to the output, the earlier ones theirs.
        y = baseline.naive_selective_scan(x, dt, A, one, one, softplus=True)
        (g,) = torch.autograd.grad(y[0, T, 0], dt)
        want = torch.sigmoid(dt.detach()) * (torch.arange(dt.shape[1]) <= T)[None, :, None]
        torch.testing.assert_close(g, want, rtol=1e-14, atol=0.0)


def test_eight_bits_of_no_channels():
    """A row without values is a row of zeros: its scale is 1."""
    x = torch.zeros(2, 3, 0)
    q, scale, total = rms_norm(x, torch.zeros(0), x, quant=torch.int8)
    assert q.shape == x.shape and total.shape == x.shape and torch.equal(scale, torch.ones(2, 3))


ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

# Stands in for the runtime's launch: notes what is asked for, launches nothing.
RECORDER = """
#include <stdint.h>
#include <stdio.h>
#include <stddef.h>
typedef struct { uint32_t x, y, z; } dim3;
int hipGetDevice(int *device) { *device = 0; return 0; }
int hipFuncSetAttribute(const void *kernel, int what, int value) { printf("limit %p %d\\n", kernel, value); fflush(stdout); return 0; }
int hipLaunchKernel(const void *kernel, dim3 grid, dim3 block, void **args, size_t lds, void *stream)
{
    printf("launch %p %u %u %u %u %u %u %zu\\n", kernel, grid.x, grid.y, grid.z, block.x, block.y, block.z, lds);
    fflush(stdout);
    return 0;
}
"""


@pytest.fixture(scope="module")
def recorded(tmp_path_factory):
    """Runs statements in a process where launches of the library are only noted (the pointers that they get are never used): lines of
    [what, kernel, numbers ...] and of what the statements print."""
    folder = tmp_path_factory.mktemp("recorder")
    (folder / "recorder.c").write_text(RECORDER)
    subprocess.run(["gcc", "-shared", "-fPIC", "-o", str(folder / "recorder.so"), str(folder / "recorder.c")], check=True)
    head = f"""
        import ctypes
        ctypes.CDLL({str(folder / "recorder.so")!r}, mode=ctypes.RTLD_GLOBAL)
        from scanscam_amd import hip, state_space as s
        L, fake = s._lib(), 0x100000
        T = lambda token=1 << 12, group=0: s._Tokens(fake, token, token, group)
        P = s._Param(fake, 0)
        def scan(**k):
            a = s._Selective(batch=1, T=4, sequences=1, channels=64, groups=1, N=16, dtype=1, saved=fake, gA=fake, workspace=fake, workspace_bytes=1 << 60, A=P)
            for n in ("x", "dt", "B", "C", "y", "gy", "gx", "gdt", "gB", "gC"):
                setattr(a, n, T())
            for n, v in k.items():
                setattr(a, n, v)
            return a
    """

    def run(statements):
        code = textwrap.dedent(head) + textwrap.dedent(statements)
        out = subprocess.run([sys.executable, "-c", code], check=True, capture_output=True, text=True, cwd=ROOT, env={**os.environ, "PYTHONPATH": ROOT})
        return [line.split() for line in out.stdout.splitlines()]

    return run


def test_the_limit_of_shared_memory_does_not_depend_on_the_call(recorded):
    """It belongs to the process, so a call's own would be another thread's too. Once a kernel, and enough for every launch."""
    lines = recorded("""
        for N in (16, 256, 1, 40, 16):
            assert L.scanscam_selective_fwd(scan(N=N), None) == 0 and L.scanscam_selective_bwd(scan(N=N), None) == 0
            assert L.scanscam_selective_bwd(scan(N=N, T=5000, parts=4), None) == 0
            assert L.scanscam_selective_fwd(scan(N=N, T=5000, parts=4), None) == 0
            assert L.scanscam_selective_bwd(scan(N=min(N, 16), batch=600, sequences=600), None) == 0
    """)
    limits = {}
    launches = 0
    for what, kernel, *numbers in lines:
        if what == "limit":
            assert kernel not in limits
            limits[kernel] = int(numbers[0])
        else:
            launches += 1
            lds = int(numbers[6])
            assert lds <= 160 * 1024 and (lds <= 64 * 1024 or lds <= limits[kernel])
    assert len(limits) == 4 and launches > 30


@pytest.mark.parametrize("rows,channels,dtype,residual", [(4000, 3000, 1, 0), (4000, 3000, 1, 1), (5, 3000, 1, 0), (1025, 2049, 0, 1), (9999, 40, 2, 0), (4096, 9000, 1, 0), (7, 1, 0, 0)])
def test_the_norm_s_workspace_follows_from_its_sizes(recorded, rows, channels, dtype, residual):
    """Asked for before the pointers are there, it is enough for the call that has them."""
    lines = recorded(f"""
        a = s._Norm(rows={rows}, channels={channels}, x_stride={channels}, dtype={dtype}, residual_dtype={residual})
        n = L.scanscam_norm_workspace_bytes(a)
        for pointer in ("x", "residual", "sum", "gy", "gx", "gresidual", "gweight", "rstd", "workspace"):
            setattr(a, pointer, fake)
        a.weight, a.workspace_bytes = P, n
        print("rc", L.scanscam_norm_bwd(a, None), n == L.scanscam_norm_workspace_bytes(a))
        a.workspace_bytes = n - 4
        print("rc", L.scanscam_norm_bwd(a, None))
    """)
    assert [line for line in lines if line[0] == "rc"] == [["rc", "0", "True"], ["rc", "5"]]


def launches(lines):
    """(workgroups, threads of a workgroup) of each launch; every dimension of the grid has fewer than 2^32 threads, all but the first up to 65 535 workgroups."""
    out = []
    for what, _, *n in lines:
        if what == "launch":
            x, y, z, bx, by, bz, _ = map(int, n)
            assert x * bx < 1 << 32 and y <= 65535 and z == 1 and x * y > 0
            out.append((x * y, bx * by * bz))
    return out


def test_selective_scans_of_many_parts_are_several_launches(recorded):
    """Workgroups: of 32 channels (16, or two sets of them, backwards) for each sequence; none is left out and none comes twice."""
    for batch, channels in ((65536, 2048), (1 << 23, 64), (1 << 20, 65536)):
        lines = recorded(f"assert L.scanscam_selective_fwd(scan(batch={batch}, sequences={batch}, T=1, channels={channels}, N=4), None) == 0")
        assert sum(n for n, threads in launches(lines)) == batch * channels // 32
        lines = recorded(f"assert L.scanscam_selective_bwd(scan(batch={batch}, sequences={batch}, T=1, channels={channels}, N=4), None) == 0")
        assert sum(n for n, threads in launches(lines) if threads == 256) == batch * channels // 32 + batch * 8 // 1024 + (batch * 8 % 1024 > 0)
    # gradients of B and C: tokens x 2 N values, four a lane
    lines = recorded("assert L.scanscam_selective_bwd(scan(batch=1 << 20, sequences=1 << 20, T=100, channels=4, N=256), None) == 0")
    assert sum(n for n, threads in launches(lines)[:-1] if threads == 256) == (1 << 20) + (100 << 20) * 512 // 1024
    # packed: the numbers of parts that there may be
    lines = recorded("assert L.scanscam_selective_fwd(scan(batch=1, sequences=3000000, T=4000000, channels=2048, offsets=fake), None) == 0")
    assert sum(n for n, _ in launches(lines)) == 3000000 * 64
    assert recorded("print(L.scanscam_selective_fwd(scan(batch=1 << 20, sequences=1 << 20, T=1 << 11), None))") == [["1"]]  # 2^31 tokens
    assert recorded("print(L.scanscam_selective_fwd(scan(batch=1 << 25, sequences=1 << 25, T=0), None))")[-1] == ["0"]


def test_norms_of_many_rows_are_several_launches(recorded):
    for rows, channels, eight in (((1 << 26) + 3, 8, 0), ((1 << 27) + 1, 64, 17), (1 << 30, 1, 0), (1 << 25, 16384, 16), (100, 5, 0)):
        lines = recorded(f"""
            a = s._Norm(rows={rows}, channels={channels}, x_stride={channels}, dtype=1, out_dtype={eight or 1}, x=fake, y=fake, scale=fake, weight=P)
            assert L.scanscam_norm_fwd(a, None) == 0
        """)
        assert sum(n * threads // 64 for n, threads in launches(lines)) >= rows  # (a row has a wave or more)


def test_convolutions_of_many_stretches_are_several_launches(recorded):
    for batch, T, channels, packed in (((1 << 23) + 9, 1, 4, 0), (1, (1 << 30) + 5, 64, 0), (1 << 24, 3, 4096, 0), (1, 5, 4096, 1 << 26), (2, 9, 24, 0)):
        lines = recorded(f"""
            a = s._Conv(batch={batch}, T={T}, sequences={packed or batch}, channels={channels}, K=4, dtype=1, x=T(), y=T(), gy=T(), gx=T(), weight=P, gweight=fake,
                        offsets={'fake' if packed else 'None'}, state_in=fake, state_out=fake, gstate_in=fake, workspace=fake, workspace_bytes=1 << 62)
            assert L.scanscam_conv_fwd(a, None) == 0
            print("backwards", flush=True)
            assert L.scanscam_conv_bwd(a, None) == 0
        """)
        back = lines.index(["backwards"])
        for part, vec in ((lines[:back], 8), (lines[back + 1:], 4)):
            lanes = sum(n * threads for n, threads in launches(part) if threads == 256)
            assert lanes >= channels // vec * ((packed or batch) + batch * -(-T // 128))  # (a lane a vector of each state and of each stretch at least)
    assert recorded("print(L.scanscam_conv_fwd(s._Conv(batch=4, T=1 << 29, sequences=4, channels=8, K=4, x=T(), y=T(), weight=P), None))") == [["1"]]  # 2^31 tokens


def test_steps_of_many_rows_or_channels_are_several_launches(recorded):
    for rows, channels, N in ((1 << 24, 32, 16), (3, 1 << 20, 128), ((1 << 25) + 1, 8, 1), (1, 1, 1)):
        lines = recorded(f"""
            a = s._SelectiveStep(rows={rows}, channels={channels}, groups=1, N={N}, slots=1, slot=fake, state=fake, A=P)
            for n in ("x", "dt", "B", "C", "y"):
                setattr(a, n, T())
            assert L.scanscam_selective_step_fwd(a, None) == 0
        """)
        lanes = min(32, 1 << max(0, (N - 1).bit_length() - 2))
        assert sum(n for n, _ in launches(lines)) == rows * -(-channels * lanes // 256)
        lines = recorded(f"""
            a = s._ConvStep(rows={rows}, channels={channels}, K=4, slots=1, slot=fake, state=fake, weight=P, x=T(), y=T())
            assert L.scanscam_conv_step_fwd(a, None) == 0
        """)
        assert sum(n * threads for n, threads in launches(lines)) >= rows * -(-channels // 4)


def test_steps_on_the_cpu_keep_tangents():
    """Their loops are ordinary operations: what a step's input adds to its output and to the state, forwards."""
    state, w = torch.zeros(1, 2, 3), torch.rand(3, 3)
    x, tangent = torch.rand(1, 3), torch.rand(1, 3)
    A, B = -torch.rand(3, 4), torch.rand(1, 4)
    with forward_ad.dual_level():
        dual, kept = forward_ad.make_dual(x, tangent), forward_ad.make_dual(torch.zeros(1, 3, 4), torch.zeros(1, 3, 4))
        y = causal_conv_step(state.clone(), dual, w)
        assert torch.equal(forward_ad.unpack_dual(y).tangent, w[:, 2] * tangent)
        y = selective_scan_step(kept, dual, torch.ones(1, 3), A, B, B)
        torch.testing.assert_close(forward_ad.unpack_dual(y).tangent, tangent * (B * B).sum())
