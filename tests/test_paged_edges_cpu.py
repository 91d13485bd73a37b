"""Batched attention serving at its edges, without a GPU: the arithmetic that the kernels share with this
host (nmi_paged.hpp), and the host code of the C ABI and of the torch front end."""
import ctypes
import subprocess

import pytest

from nemotron_infer_amd import build

SHIM = """
#include "nmi_paged.hpp"
extern "C" {
int holds(int c0, int c1, int tokens, int t, int* place, int* bad) {
    bool b = false; int r = nmi::span_holds(c0, c1, tokens, t, place, &b); *bad = b; return r;
}
}
"""


@pytest.fixture(scope="module")
def shared(tmp_path_factory):
    d = tmp_path_factory.mktemp("edges")
    src, so = d / "shim.cpp", str(d / "libshim.so")
    src.write_text(SHIM)
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-shared", "-fPIC", f"-I{build.CSRC}", str(src), "-o", so],
                   check=True, timeout=120)
    return ctypes.CDLL(so)


EDGES = [-2 ** 31, -2 ** 31 + 1, -5, -1, 0, 1, 2, 8, 9, 10, 11, 2 ** 30, 2 ** 31 - 1]


def test_a_row_is_only_of_a_sequence_whose_cut_offsets_hold_it(shared):
    place, bad = ctypes.c_int(), ctypes.c_int()
    for tokens in (1, 10, 2 ** 31 - 1):
        for c0 in EDGES:
            for c1 in EDGES:
                first, end = min(max(c0, 0), tokens), min(max(c1, 0), tokens)
                for t in sorted({0, min(8, tokens - 1), min(9, tokens - 1), tokens - 1}):
                    got = shared.holds(c0, c1, tokens, t, ctypes.byref(place), ctypes.byref(bad))
                    assert bool(got) == (first <= t < end), (c0, c1, tokens, t)
                    assert not got or place.value == t - first
                    assert bool(bad.value) == (not 0 <= c0 <= c1 <= tokens)
