"""Loads that rely on a buffer descriptor's end: their whole offset is the vector one, which the hardware compares with the end.
A scalar offset is not part of that comparison on every target, so it stays 0 in the sources."""
from __future__ import annotations

import glob
import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "attention-lab_amd", "csrc")
LOAD = re.compile(r"__builtin_amdgcn_(?:raw|struct)_(?:ptr_)?buffer_(load|store)\w*\s*\(")


def arguments(text: str, at: int) -> list:
    """The arguments of the call whose opening parenthesis ends at `at`."""
    parts, depth, start = [], 0, at
    for i in range(at, len(text)):
        c = text[i]
        if c in "([{":
            depth += 1
        elif c in ")]}" and depth:
            depth -= 1
        elif c == "," and not depth or c == ")":
            parts.append(text[start:i].strip())
            start = i + 1
            if c == ")":
                return parts
    raise AssertionError("a call without an end")


def calls():
    for path in sorted(glob.glob(os.path.join(CSRC, "*.h*"))):
        with open(path) as f:
            text = f.read()
        for m in LOAD.finditer(text):
            yield pytest.param(m.group(0), arguments(text, m.end()), id=f"{os.path.basename(path)}:{text[:m.start()].count(chr(10)) + 1}")


def test_arguments():
    text = "f(r, g(a, b[1, 2]), {0, 1}, 3);"
    assert arguments(text, 2) == ["r", "g(a, b[1, 2])", "{0, 1}", "3"]
    assert len(list(calls())) >= 8


@pytest.mark.parametrize("name,args", calls())
def test_no_scalar_offset(name, args):
    # to LDS: descriptor, LDS address, size, vector offset, scalar offset, ...; else descriptor, vector offset, scalar offset, ...
    # (a store's value comes first)
    assert args[4 if "load_lds" in name else 3 if "store" in name else 2] == "0", args
