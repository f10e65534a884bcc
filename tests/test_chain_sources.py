"""Kernels that may start while the kernel before them is running must not read through the read-only path, which
promises memory that nobody writes while they are resident."""
import os
import re

import pytest

from futhark_b200 import build

SOURCES = [f for f in sorted(os.listdir(build.CSRC)) if f.endswith((".cu", ".cuh"))]


def code(name):
    with open(os.path.join(build.CSRC, name)) as f:
        return re.sub(r"//[^\n]*|/\*.*?\*/", "", f.read(), flags=re.S)


def read_only_helpers():
    """Device functions of the headers whose loads take the read-only path."""
    found = set()
    for name in SOURCES:
        if name.endswith(".cuh"):
            for fn, body in re.findall(r"\b(\w+)\(const [^)]*\)\s*\{(.*?)\n\}", code(name), flags=re.S):
                if re.search(r"ld\.global[\w:.]*\.nc|__ldg\(", body):
                    found.add(fn)
    return found


def test_the_helpers_are_recognised():
    assert "ld_stream_v4" in read_only_helpers() and "ld_chain_v4" not in read_only_helpers()


@pytest.mark.parametrize("name", [f for f in SOURCES if f.endswith(".cu") and "chain_wait();" in code(f)])
def test_kernels_of_chains_do_not_use_the_read_only_path(name):
    src = code(name)
    used = [w for w in ["__ldg", "__restrict__"] + sorted(read_only_helpers()) if re.search(r"\b%s\b" % w, src)]
    if re.search(r"ld\.global[\w:.]*\.nc", src):
        used.append("ld.global.nc")
    assert not used
