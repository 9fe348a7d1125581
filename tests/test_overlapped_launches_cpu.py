"""Kernels that may start before the kernel in front of them ends read global
memory by coherent loads: their inputs may be written while they already run, so
the read-only path (__ldg) is not theirs.  Checked in the sources."""
import re
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parents[1] / "packr_b200" / "csrc"
# every kernel that launch_overlapped (or, for the GEMV, its own launch) starts
# early, and the device helpers that load for it
PARTS = [("layer_norm.cu", n) for n in ("load_vector", "struct Rows", "fwd_kernel", "bwd_kernel", "reduce_cols_kernel")]
PARTS += [("skinny_mma.cu", n) for n in ("skinny_mma_kernel", "skinny_mma_reduce_kernel")]
PARTS += [("skinny.cu", n) for n in ("skinny_kernel", "skinny_reduce_epi_kernel")]
PARTS += [("gemv.cu", n) for n in ("struct WVec<8>", "struct WVec<4>", "struct WVec<2>", "gemv_cluster_kernel")]


def body(text, name):
    """The braces' contents of the definition of `name`."""
    at = re.search(r"\b" + re.escape(name) + r"(\s*\(|\s*\{)", text)
    assert at, name
    i = text.index("{", at.end() - 1)
    depth, j = 0, i
    while True:
        depth += (text[j] == "{") - (text[j] == "}")
        j += 1
        if depth == 0:
            return text[i:j]


@pytest.mark.parametrize("file,name", PARTS)
def test_loads_are_coherent(file, name):
    code = body((CSRC / file).read_text(), name)
    code = re.sub(r"//[^\n]*", "", code)
    bad = re.findall(r"__ldg\(|\bload_io\(|ld\.global\.nc", code)
    assert not bad, (file, name, bad)


def test_every_overlapped_kernel_is_in_the_list():
    known = {n for _, n in PARTS}
    for f in CSRC.glob("*.cu"):
        text = f.read_text()
        for kern in re.findall(r"return launch_overlapped\(\s*(\w+)|= launch_overlapped\(\s*(\w+)", text):
            name = kern[0] or kern[1]
            if name == "kern":  # layer_norm.cu: `auto kern = ragged ? X<..> : X<..>`
                names = re.findall(r"auto kern = s\.ragged \? (\w+)<", text)
                assert names and set(names) <= known, f.name
            else:
                assert name in known, (f.name, name)
