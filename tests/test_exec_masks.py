"""CPU: the built kernels' code where lanes that went apart come together again. A block that a branch
for no lanes (s_cbranch_execz) goes to, or that stands behind a loop's branch for some (s_cbranch_execnz), begins by
giving the others back to the mask:

    s_or_b64 exec, exec, ...

A copy of a vector register or a spill in front of that is done for some lanes only, while the code behind uses it for
all: the compiler has put copies there in a kernel short of registers (lanes without a row of x lost
their thread's index, and rows of the result were not stored). Lane writes and scalar instructions go by no mask."""
import os
import re
import subprocess

import pytest

import pyc_amd.build as build

OBJDUMP = os.path.join(build.ROCM, "llvm", "bin", "llvm-objdump")
NO_MASK = re.compile(r"s_|v_readlane|v_readfirstlane|v_writelane")


def code_objects(path):
    """The gfx950 code objects in the bundles of a library."""
    with open(path, "rb") as f:
        data = f.read()
    for m in re.finditer(b"__CLANG_OFFLOAD_BUNDLE__", data):
        at, n = m.start(), int.from_bytes(data[m.end():m.end() + 8], "little")
        p = m.end() + 8
        for _ in range(n):
            offset, size, length = (int.from_bytes(data[p + 8 * i:p + 8 * i + 8], "little") for i in range(3))
            name = data[p + 24:p + 24 + length]
            p += 24 + length
            if name.endswith(build.ARCH.encode()) and size:
                yield data[at + offset:at + offset + size]


def early(lines):
    """(kernel, instruction) of every masked vector instruction between the beginning of such a block and the
    mask's restoration there, and how many restorations there are. Blocks that do not restore it are left alone."""
    text, kernel = [], None
    targets = set()
    for line in lines:
        m = re.match(r"[0-9a-f]+ <(\w+)>:", line)
        if m:
            kernel = m[1]
            continue
        m = re.match(r"\s+([sv]_\S+|ds_\S+|global_\S+|scratch_\S+|buffer_\S+|flat_\S+)\s*(.*?)\s*// ([0-9A-F]+):", line)
        if not m:
            continue
        text.append((kernel, int(m[3], 16), m[1], m[2]))
        t = re.search(r"<(\w+)\+0x([0-9a-f]+)>", line)
        if m[1] == "s_cbranch_execz" and t:
            targets.add((t[1], int(t[2], 16)))
    first = {}
    for kernel, at, _, _ in text:
        first.setdefault(kernel, at)
    ends = {"s_endpgm", "s_branch", "s_barrier", "s_setpc_b64"}
    found, joins = [], 0
    for i, (kernel, at, _, _) in enumerate(text):
        if (kernel, at - first[kernel]) not in targets and (i == 0 or text[i - 1][2] != "s_cbranch_execnz"):
            continue
        held = []
        for _, _, op, args in text[i:i + 200]:
            if op == "s_or_b64" and args.startswith("exec, exec"):
                joins += 1
                found += [(kernel, f"{o} {a}") for o, a in held]
                break
            if op in ends or op.startswith("s_cbranch") or "saveexec" in op or "exec" in args.split(",")[0]:
                break
            if not NO_MASK.match(op):
                held.append((op, args))
    return found, joins


@pytest.mark.skipif(not os.path.exists(OBJDUMP), reason="no llvm-objdump")
def test_nothing_before_the_mask_is_back(tmp_path):
    path = build.LIB_PATH
    if not os.path.exists(path):
        build.build()
    joins = n = 0
    for n, obj in enumerate(code_objects(path), 1):
        f = tmp_path / f"{n}.co"
        f.write_bytes(obj)
        out = subprocess.run([OBJDUMP, "-d", str(f)], stdout=subprocess.PIPE, text=True, check=True).stdout
        found, j = early(out.splitlines())
        joins += j
        assert not found, found[:5]
    assert n == len(build.sources()[0]) and joins > 1000


def test_the_rule_by_hand():
    code = """0000000000001000 <k>:
	s_and_saveexec_b64 s[14:15], vcc                           // 000000001000: BE8E206A
	s_cbranch_execz 2                                          // 000000001004: BF880002 <k+0x10>
	v_mov_b32_e32 v7, -1                                       // 000000001008: 7E0E02C1
	s_mov_b32 s1, 0                                            // 00000000100C: BE810080
	%s                                                         // 000000001010: 7ECC03B6
	s_or_b64 exec, exec, s[14:15]                              // 000000001014: 87FE0E7E
"""
    assert early((code % "v_mov_b32_e32 v102, v182").splitlines()) == ([("k", "v_mov_b32_e32 v102, v182")], 1)
    assert early((code % "scratch_load_dword v0, off, off").splitlines())[0]
    assert early((code % "v_writelane_b32 v255, s66, 13").splitlines()) == ([], 1)
    assert early((code % "s_nop 0").splitlines()) == ([], 1)
