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
int look_on(unsigned at, unsigned upto, int b0, int batch) { return nmi::look_on(at, upto, b0, batch); }
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


@pytest.mark.parametrize("batch", [1, 64, 65, 128, 129, 1000])
def test_the_search_for_a_tile_ends_within_the_batch(shared, batch):
    """As the decode kernel looks for the sequence of a tile, 64 lengths at a time: also where they have
    become less, or nothing, since the tiles were dealt, it ends and stays within the batch."""
    was = [3 + b % 5 for b in range(batch)]
    for now in (was, [0] * batch, [1] * batch, was[:batch // 2] + [0] * (batch - batch // 2)):
        for at in (0, 1, sum(now) - 1, sum(now), sum(was) - 1, 2 ** 32 - 1):
            if at < 0:
                continue
            b0, steps, upto = 0, 0, sum(now[:64])
            while shared.look_on(ctypes.c_uint(at), ctypes.c_uint(upto), b0, batch):
                b0, steps = b0 + 64, steps + 1
                assert b0 < batch and steps <= batch // 64
                upto += sum(now[b0:b0 + 64])
            if at < sum(now):
                assert upto - sum(now[b0:b0 + 64]) <= at < upto
            else:
                assert b0 == (batch - 1) // 64 * 64
