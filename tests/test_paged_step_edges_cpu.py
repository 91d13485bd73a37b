"""A serving step on a paged cache without a GPU, where it is easiest to get wrong: loops whose ends come from lengths in
device memory, counts past a type's range."""
import ctypes
import subprocess

import pytest
import torch

from nemotron_infer_amd import build, ops

SHIM = """
#include "nmi_paged.hpp"
extern "C" unsigned back(unsigned total, int count, int n_pages, int* bad) {
    bool b = false; unsigned r = nmi::pages_back(total, count, n_pages, &b); *bad = b; return r;
}
"""


@pytest.fixture(scope="module")
def hpp(tmp_path_factory):
    d = tmp_path_factory.mktemp("edges")
    src, so = d / "shim.cpp", str(d / "libshim.so")
    src.write_text(SHIM)
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-shared", "-fPIC", f"-I{build.CSRC}", str(src), "-o", so],
                   check=True, timeout=120)
    so = ctypes.CDLL(so)
    so.back.restype = ctypes.c_uint
    return so


def test_pages_that_come_back_end_with_the_room_for_them(hpp):
    """Whatever lengths claim (64 sequences of 2^26 pages each are more than 32 bits count): no more than the stack
    holds, so that a thread's counter, 1024 at a time, passes the end without a wrap."""
    most = 2 ** 31 - 1
    for n_pages in (1, 5, 1000, 2 ** 20, most):
        for count in {0, 1, n_pages // 2, n_pages - 1, n_pages}:
            for total in (0, 1, 4, 999, 2 ** 20, 2 ** 31 - 1, 2 ** 31, 2 ** 32 - 1024, 2 ** 32 - 1):
                bad = ctypes.c_int()
                got = hpp.back(total, count, n_pages, ctypes.byref(bad))
                assert got == min(total, n_pages - count) and bool(bad.value) == (total > n_pages - count)
                assert got + 1024 < 2 ** 32 and count + got <= n_pages


@pytest.mark.parametrize("tokens", [2 ** 31, 2 ** 40, 2 ** 62, 2 ** 63 - 1, -1])
def test_front_end_refuses_rows_past_the_type_before_it_asks_for_memory(tokens):
    """As a count out of range, not as memory that cannot be had."""
    ints = lambda *s: torch.zeros(*s, dtype=torch.int32)  # noqa: E731
    with pytest.raises(ValueError, match=f"tokens={tokens} is out of range"):
        ops.kv_assign_paged(ints(3), ints(3), ints(3, 4), ints(9), ints(1), 16, tokens=tokens)
    with pytest.raises((ValueError, TypeError), match="tokens"):
        ops.kv_assign_paged(ints(3), ints(3), ints(3, 4), ints(9), ints(1), 16, tokens=2 ** 64)
