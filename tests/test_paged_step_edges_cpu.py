"""A serving step on a paged cache without a GPU, where it is easiest to get wrong: loops whose ends come from lengths in
device memory, counts past a type's range, what rounded bounds promise."""
import ctypes
import subprocess

import numpy as np
import pytest
import torch

from nemotron_infer_amd import _lib, build, ops
from oracle import block, e4m3, paged
from tests.test_host_runtime_cpu import host  # noqa: F401  (a fixture)

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


def _stored_bounds(keys):
    """As the operator stores them: of float32 keys, rounded to the nearest bf16."""
    bits = block.bf16_round_exact(paged.page_bounds(keys.astype(np.float32).astype(np.float64)))
    return (bits.astype(np.uint32) << 16).view(np.float32).astype(np.float64)


def test_bounds_as_they_are_stored_bound_the_keys():
    """Of bf16 keys, and of codes under powers of two from 2^-124 to 2^119, the stored bounds are the keys' own, so that no
    key's product passes the score; under other scales they may lie 2^-8 of their value inside."""
    rng = np.random.default_rng(8)
    lut = e4m3.decode_lut()
    codes = lut[np.isfinite(lut)][rng.integers(0, 254, (6, 2, 32, 128))]
    bf16 = rng.integers(0, 0x7F80, (6, 2, 32, 128)) | rng.integers(0, 2, (6, 2, 32, 128)) << 15
    exact = [(bf16.astype(np.uint32) << 16).view(np.float32).astype(np.float64)]
    exact += [codes * 2.0 ** e for e in (-124, -60, -7, 0, 5, 60, 119)]
    for keys in exact:
        bounds = _stored_bounds(keys)
        assert np.array_equal(bounds, paged.page_bounds(keys))
    q = rng.standard_normal((2, 128))
    short = 0
    for scale in (0.01, 0.0371, 1.7, 2.0 ** -7 * 1.001):
        keys = (codes.astype(np.float32) * np.float32(scale)).astype(np.float64)
        bounds = _stored_bounds(keys)
        lo, hi = bounds[:, :, 0], bounds[:, :, 1]
        true = paged.page_bounds(keys)
        assert (np.abs(bounds - true) <= 2.0 ** -8 * np.abs(true)).all()
        short += int((hi < true[:, :, 1]).sum() + (lo > true[:, :, 0]).sum())
        for g in range(2):
            up, down = np.maximum(q[g], 0), np.minimum(q[g], 0)
            score = (hi[:, g] * up + lo[:, g] * down).sum(-1)
            slack = 2.0 ** -8 * (np.abs(true[:, g, 1]) * up - np.abs(true[:, g, 0]) * down).sum(-1)
            assert ((keys[:, g] @ q[g]).max(-1) <= score + slack + 1e-9 * np.abs(score)).all()
    assert short > 100                                   # (they do lie inside: the bound is no bound there)


def test_keys_may_stand_for_values_in_the_bounds_and_not_be_left_out(host):  # noqa: F811
    """The values are not read, and checked as elsewhere."""
    got = host("""
W, ST = 1 << 38, 1 << 12
result = []
for v, vs in ((W, W), (None, W), (W, None)):
    c = _lib.PagedKv(W, v, 8 * 16 * 128, 16 * 128, 128, W, 64, W, vs, 2, 100, 16, 64, 8)
    result.append([L.nmi_kv_bounds_paged(ctypes.addressof(c), W, None, W, 3, 3, ST), len(launches())])
""")
    assert got == [[0, 1], [_lib.NMI_ERR_INVALID_ARG, 0], [_lib.NMI_ERR_INVALID_ARG, 0]]


def test_the_places_alone_cost_a_launch_where_all_pages_are_attended(host):  # noqa: F811
    got = host("""
W, ST = 1 << 38, 1 << 12
result = []
for selected in (None, W):
    c = _lib.PagedKv(W, W, 8 * 64 * 128, 64 * 128, 128, W, 64, W, W, 2, 100, 64, 64, 8)
    need = L.nmi_sdpa_decode_paged_sparse_workspace_bytes(2, 40, 8, 64, 64)
    rc = L.nmi_sdpa_decode_paged_sparse(ctypes.addressof(c), W, 5120, W, 5120, W, W, 64, selected, 2, 40, 0.1, W, need, ST)
    result.append([rc, [l[0] for l in launches()]])
""")
    (rc, decode), (rc_selected, with_places) = got
    assert rc == rc_selected == 0 and with_places[1:] == decode and "page_select" in with_places[0]
