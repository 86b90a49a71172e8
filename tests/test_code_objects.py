"""
The library's kernels as they were compiled, read from the built file. No GPU is needed.

Where a part of a wave's lanes has gone through a branch or a loop the others wait at a join, whose code makes the mask of lanes (EXEC) whole again. What is written to a
vector register between the join's first instruction and that is written for no lanes, or for some: the compiler has put copies of registers there in kernels that keep scalar
registers in lanes of vector ones (a wave's number of each lane, of which addresses were made: an access out of range). No kernel may have one.
"""
import os
import re
import shutil
import subprocess

import pytest

from scanscam_amd import hip

OBJDUMP = "/opt/rocm/llvm/bin/llvm-objdump"
WRITES = re.compile(r"v_(?!writelane|readlane|readfirstlane|cmp|nop)|scratch_load|global_load|ds_read|buffer_load|flat_load")
EXEC = re.compile(r"s_\w+_saveexec|s_\w+ exec|v_cmpx")
END = re.compile(r"s_(c?branch|endpgm|setpc)")


def functions(text):
    """(name, [(address, instruction, address that it branches to or None)])"""
    name, out = None, []
    for line in text.splitlines():
        head = re.match(r"([0-9a-f]+) <(\S+)>:", line)
        if head:
            if name:
                yield name, out
            name, out, start = head.group(2), [], int(head.group(1), 16)
            continue
        got = re.match(r"\s+(\S.*?)\s+// ([0-9A-F]+):", line)
        if got and name:
            to = re.search(r"<\S+?\+0x([0-9a-f]+)>", line)
            out.append((int(got.group(2), 16), got.group(1), start + int(to.group(1), 16) if to else None))
    if name:
        yield name, out


def early_writes(code):
    """Writes to vector registers at joins before the mask is whole."""
    at = {address: i for i, (address, _, _) in enumerate(code)}
    joins = []
    for i, (_, text, to) in enumerate(code):
        # (right behind what leaves lanes out: elsewhere such a branch is one that is always, or never, taken)
        if text.startswith("s_cbranch_exec") and any(EXEC.match(code[k][1]) for k in range(max(i - 3, 0), i)):
            joins.append(at.get(to) if text.startswith("s_cbranch_execz") else i + 1)  # (behind a loop no lane is left)
    joins = [i for i in joins if i is not None]
    for first in sorted(set(joins)):
        writes = []
        for address, text, _ in code[first:]:
            if re.match(r"s_or_b64 exec, exec", text):
                yield from writes
            if END.match(text) or EXEC.match(text):
                break
            if WRITES.match(text):
                writes.append(f"{address:x}: {text}")


def test_the_search_finds_what_it_looks_for():
    code = [(0, "s_and_saveexec_b64 s[4:5], vcc", None), (4, "s_cbranch_execz 3", 20), (8, "v_add_u32_e32 v1, v2, v1", None), (12, "s_andn2_b64 exec, exec, s[0:1]", None), (16, "s_cbranch_execnz 65533", 8),
            (20, "v_writelane_b32 v9, s1, 3", None), (24, "v_mov_b32_e32 v3, v4", None), (28, "s_or_b64 exec, exec, s[4:5]", None), (32, "v_mov_b32_e32 v5, v6", None), (36, "s_endpgm", None)]
    assert list(early_writes(code)) == ["18: v_mov_b32_e32 v3, v4"]
    assert not list(early_writes(code[:6] + code[7:]))


def test_no_kernel_writes_registers_before_its_mask_is_whole(tmp_path):
    if not os.path.exists(OBJDUMP):
        pytest.skip("no llvm-objdump")
    lib = shutil.copy(hip.LIB_PATH, tmp_path / "lib.so")
    subprocess.run([OBJDUMP, "--offloading", lib], check=True, cwd=tmp_path, capture_output=True)
    objects = sorted(p for p in tmp_path.iterdir() if "gfx950" in p.name)
    assert objects
    running = [subprocess.Popen([OBJDUMP, "-d", "--no-show-raw-insn", str(p)], stdout=subprocess.PIPE, text=True) for p in objects]
    kernels, found = 0, []
    for p in running:
        for name, code in functions(p.communicate()[0]):
            kernels += 1
            found += [(name, w) for w in early_writes(code)]
        assert p.returncode == 0
    assert kernels > 100 and not found, (len(found), found[:5])
