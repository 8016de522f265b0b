"""CPU: how the kernels keep loads inside their arrays. A descriptor covers its array for all of a
kernel's steps; what is past the end (a step behind the last, k past K, a row that there is not) is
kept out by the lane's own offset, the one part of an address that the range check surely has. So no
byte count of a descriptor depends on where in a loop a kernel is: those would rest on how the check
takes a scalar offset against the smaller count."""
import glob
import os
import re

import pytest

KERNELS = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "pyc_amd", "csrc", "kernels")
CALL = re.compile(r"make_buf(?:fer)?_rsrc\(")


def _arguments(text, at):
    """The text between the parenthesis that opens at `at` and the one that closes it."""
    depth = 0
    for i in range(at, len(text)):
        depth += {"(": 1, ")": -1}.get(text[i], 0)
        if depth == 0:
            return text[at + 1:i]
    raise AssertionError("no end")


def _chosen_by_comparison(arguments):
    return re.search(r"[<>]", re.sub(r"\w+_cast<[^<>]*>", "", arguments)) is not None


def _descriptors(text):
    return [_arguments(text, m.end() - 1) for m in CALL.finditer(text)]


@pytest.mark.parametrize("name", sorted(os.path.basename(f) for f in glob.glob(os.path.join(KERNELS, "*.hip"))))
def test_byte_counts_hold_for_every_step(name):
    with open(os.path.join(KERNELS, name)) as f:
        for d in _descriptors(f.read()):
            assert not _chosen_by_comparison(d), d


def test_the_rule_by_hand():
    text = "make_buffer_rsrc(p, 0, i < chunks ? wbytes : 0u, 0x00020000); make_buf_rsrc(static_cast<const char*>(g.w) + e, n)"
    assert [_chosen_by_comparison(d) for d in _descriptors(text)] == [True, False]
