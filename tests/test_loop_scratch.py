"""CPU: the kernels of the products by expert that are short of registers (256 x 256 tiles, 128 x 256 tiles with 4-bit weights)
keep values of a tile's start and end in scratch, and none of their loops over K. Looked up in the built library: a
loop over K is an innermost loop with matrix instructions."""
import os
import re
import subprocess

import pytest

import pyc_amd.build as build
from tests.test_exec_masks import OBJDUMP, code_objects

LINE = re.compile(r"\s+([a-z]\w+)\s*(.*?)\s*// ([0-9A-F]+):")


def loops(lines):
    """{kernel: [instructions of an innermost loop]} of the loops with matrix instructions."""
    code, kernel = {}, None
    for line in lines:
        m = re.match(r"[0-9a-f]+ <(\w+)>:", line)
        if m:
            kernel = m[1]
            continue
        m = LINE.match(line)
        if m and kernel:
            t = re.search(r"<\w+\+0x([0-9a-f]+)>", line) if m[1].startswith(("s_cbranch", "s_branch")) else None
            code.setdefault(kernel, []).append((int(m[3], 16), m[1], int(t[1], 16) if t else None))
    found = {}
    for kernel, text in code.items():
        first, place = text[0][0], {at: i for i, (at, _, _) in enumerate(text)}
        spans = sorted((place[first + to], i) for i, (at, _, to) in enumerate(text) if to is not None and first + to <= at)
        for a, b in spans:
            ops = [op for _, op, _ in text[a:b + 1]]
            if not any(a <= c and d <= b and (c, d) != (a, b) for c, d in spans) and sum("mfma" in op for op in ops) >= 4:
                found.setdefault(kernel, []).append(ops)
    return found


@pytest.mark.skipif(not os.path.exists(OBJDUMP), reason="no llvm-objdump")
def test_no_scratch_in_loops_over_k(tmp_path):
    if not os.path.exists(build.LIB_PATH):
        build.build()
    seen = {}
    for n, obj in enumerate(code_objects(build.LIB_PATH)):
        if b"grouped_" not in obj:
            continue
        f = tmp_path / f"{n}.co"
        f.write_bytes(obj)
        out = subprocess.run([OBJDUMP, "-d", str(f)], stdout=subprocess.PIPE, text=True, check=True).stdout
        for kernel, each in loops(out.splitlines()).items():
            for ops in each:
                assert not any(op.startswith("scratch_") for op in ops), kernel
            seen[kernel] = len(each)
    # two types; a loop for each height of a tile (the streamed kernels' loops hold others, and those kernels no scratch)
    tiles = {k: v for k, v in seen.items() if "grouped_tile" in k}
    assert len(tiles) == 8 and all(v >= 3 for v in tiles.values())
    assert sum("grouped_w4_tile" in k for k in seen) == 48 and sum("grouped_ring" in k for k in seen) == 8


def test_loops_by_hand():
    code = """0000000000001000 <k>:
	scratch_load_dword v0, off, off                            // 000000001000: DC
	v_mfma_f32_16x16x32_bf16 v[0:3], v[4:7], v[8:11], v[0:3]   // 000000001008: D3
	v_mfma_f32_16x16x32_bf16 v[0:3], v[4:7], v[8:11], v[0:3]   // 000000001010: D3
	v_mfma_f32_16x16x32_bf16 v[0:3], v[4:7], v[8:11], v[0:3]   // 000000001018: D3
	%s                                                         // 000000001020: D3
	s_cbranch_scc1 65528                                       // 000000001028: BF <k+0x8>
	s_cbranch_vccnz 65526                                      // 00000000102C: BF <k>
	s_endpgm                                                   // 000000001030: BF
"""
    mfma = "v_mfma_f32_16x16x32_bf16 v[0:3], v[4:7], v[8:11], v[0:3]"
    (ops,) = loops((code % mfma).splitlines())["k"]
    assert ops == ["v_mfma_f32_16x16x32_bf16"] * 4 + ["s_cbranch_scc1"]
    assert loops((code % "scratch_load_dword v0, off, off").splitlines()) == {}
