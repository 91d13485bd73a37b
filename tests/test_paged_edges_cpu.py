"""Batched attention serving at its edges, without a GPU: the arithmetic that the kernels share with this
host (nmi_paged.hpp), and the host code of the C ABI and of the torch front end."""
import ctypes
import json
import os
import subprocess
import sys

import numpy as np
import pytest
import torch

from nemotron_infer_amd import build, ops
from tests.conftest import ROOT
from tests.test_host_runtime_cpu import PRELUDE

SHIM = """
#include <cmath>
#include "nmi_paged.hpp"
extern "C" {
int holds(int c0, int c1, int t) { return nmi::span_holds(c0, c1, t); }
int place(int c0, int t) { return nmi::span_place(c0, t); }
int span(int c0, int c1, int tokens, int* first) { bool b = false; return nmi::checked_span(c0, c1, tokens, first, &b); }
void turns(const double* f, long n, float* got, float* want) {
    for (long i = 0; i < n; ++i) {
        nmi::cos_sin(f[i], &got[2 * i], &got[2 * i + 1]);
        const long double a = 6.283185307179586476925286766559L * f[i];
        want[2 * i] = (float)cosl(a), want[2 * i + 1] = (float)sinl(a);
    }
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
    first = ctypes.c_int()
    for tokens in (1, 10, 2 ** 31 - 1):
        for c0 in EDGES:
            for c1 in EDGES:
                n = shared.span(c0, c1, tokens, ctypes.byref(first))
                for t in sorted({0, min(8, tokens - 1), min(9, tokens - 1), tokens - 1}):
                    got = shared.holds(c0, c1, t)
                    assert bool(got) == (first.value <= t < first.value + n), (c0, c1, tokens, t)
                    assert not got or shared.place(c0, t) == t - first.value


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


# The stand-in for the HIP runtime of test_host_runtime_cpu.py, which also says where the library's host
# memory is: one allocation, of an error word for each kind (a GEMM's, a paged call's) and device (64).
WORDS_STUB = """
#define hipHostMalloc plain_hipHostMalloc
#include "hip_host_stub.cpp"
#undef hipHostMalloc
static void* g_host = nullptr;
extern "C" int hipHostMalloc(void** p, size_t bytes, unsigned flags) {
    if (g_host || bytes != 2 * 64 * 4) std::abort();
    const int rc = plain_hipHostMalloc(p, bytes, flags);
    g_host = *p;
    return rc;
}
extern "C" uint32_t* stub_host_memory() { return static_cast<uint32_t*>(g_host); }
"""

WORDS_BODY = """
hip.stub_host_memory.restype = ctypes.POINTER(ctypes.c_uint32)
W, ST = 1 << 38, 1 << 12
c = _lib.PagedKv(W, W, 8 * 16 * 128, 16 * 128, 128, W, 64, None, None, 0, 100, 16, 64, 8)
def decode():
    return L.nmi_sdpa_decode_paged(ctypes.addressof(c), W, 5120, W, 5120, W, 2, 40, 0.1, W, 1 << 30, ST)
def append():
    return L.nmi_kv_append_paged(ctypes.addressof(c), None, 0, W, 1024, W, 1024, None, 0, None, 0, None, W, 2, 2, 0, None, 0, 0, ST)
def prefill():
    return L.nmi_sdpa_prefill_packed_bf16(W, 5120, W, 1024, W, 1024, W, 5120, W, 2, 300, 40, 8, 0.1, ST)
def linear():
    return L.nmi_linear_fp8_w8a16(W, 3136, W, 3136, W, W, 3136, 1, 3136, 3136, ST)
def gemv():
    return L.nmi_gemv_fp8(W, W, W, W, 3136, 3136, ST)
def mlp():
    return L.nmi_mlp_forward_fp8(W, W, W, W, W, W, W, 1, 3136, 12544, 1e-5, W, 1 << 30, ST)
def attn():
    return L.nmi_attn_forward_fp8(W, W, W, W, W, W, W, W, W, W, W, 520, W, W, 520, 3136, 40, 8, 1e-5, W, 1 << 32, ST)
gemm_side, paged_side = [linear, gemv, mlp, attn], [append, decode, prefill]
for f in gemm_side + paged_side:
    assert f() == 0, L.nmi_last_error()
words = hip.stub_host_memory()
GEMM, PAGED = 0, 64
result = []
for kind, mine, others in ((GEMM, gemm_side, paged_side), (PAGED, paged_side, gemm_side)):
    for f in mine:
        words[kind] = 1
        hip.stub_take_log()
        other = [g() for g in others]
        ran = len(launches())
        got = [f(), len(launches()), L.nmi_last_error().decode(), f()]
        result.append([kind, other, ran, got])
    for status in (L.nmi_async_status, L.nmi_sync):
        words[kind] = 1
        result.append([kind, [0], 1, [status(), 0, L.nmi_last_error().decode(), status()]])
words[GEMM] = words[PAGED] = 1
result.append([sorted([L.nmi_async_status(), L.nmi_async_status()]), L.nmi_async_status(), words[GEMM], words[PAGED]])
"""


def test_an_operators_error_is_returned_to_calls_of_its_kind(tmp_path):
    """Bad device data of a paged call is reported to the next call on a paged cache or packed prompts and by
    the status entries, once; linears and blocks are not refused for it, and a GEMM's error not taken
    by the paged entries."""
    (tmp_path / "words.cpp").write_text(WORDS_STUB)
    stub = str(tmp_path / "libwords.so")
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-shared", "-fPIC", f"-I{os.path.join(ROOT, 'tests')}",
                    str(tmp_path / "words.cpp"), "-o", stub], check=True, timeout=120)
    code = PRELUDE.format(stub=stub) + WORDS_BODY + "\nprint(json.dumps(result))\n"
    r = subprocess.run([sys.executable, "-c", code], cwd=ROOT, capture_output=True, text=True, timeout=120)
    assert r.returncode == 0, r.stderr
    *cases, both = json.loads(r.stdout.splitlines()[-1])
    assert len(cases) == 4 + 3 + 4
    for kind, other, ran, (rc, launched, why, again) in cases:
        assert other == [0] * len(other) and ran >= len(other), (kind, other, ran)
        assert rc == -6 and launched == 0 and again == 0
        assert ("page" in why) == (kind == 64) and ("stream-K" in why) == (kind == 0)
    assert both == [[-6, -6], 0, 0, 0]


def test_the_rotations_sine_and_cosine_are_rounded_once(shared):
    """Against the long double functions rounded to float32.  An error of up to 2^-48 before the rounding (the
    polynomials' 2e-15 and some 64-bit roundings), to either side, crosses the middle of two floats, which are
    2^-24 of the value apart at least, for 2^-23 of the values: 0.5 of the 4 million here."""
    rng = np.random.default_rng(70)
    f = np.concatenate([rng.uniform(-0.5, 0.5, 2_000_000), rng.uniform(-1, 1, 1000) * 2.0 ** rng.integers(-60, -2, 1000)])
    f = np.concatenate([f, [0.0, -0.0]])
    got, want = np.empty((len(f), 2), np.float32), np.empty((len(f), 2), np.float32)
    at = lambda x: x.ctypes.data_as(ctypes.c_void_p)  # noqa: E731
    shared.turns(at(f), ctypes.c_long(len(f)), at(got), at(want))
    off = got != want
    assert off.sum() <= 3 and np.array_equal(got[off], np.nextafter(want[off], got[off]))
    # the quarters and eighths of a turn, whose small sine or cosine is what 64 bits of 2 pi make of it
    f = np.arange(-4, 5) / 8
    got, want = got[:9], want[:9]
    shared.turns(at(f), ctypes.c_long(9), at(got), at(want))
    assert np.abs(got.astype(np.float64) - want).max() <= 2.0 ** -24


def test_strides_of_dimensions_of_one_element_have_no_meaning():
    """K and V of one KV head made in either order of heads and positions, and a page table of one page per
    sequence whatever its column stride: valid (here refused only for not being on a GPU); strides that do
    mean something still have to agree."""
    k = torch.zeros(5, 1, 16, 128, dtype=torch.bfloat16)
    v = torch.zeros(5, 16, 1, 128, dtype=torch.bfloat16).transpose(1, 2)
    assert k.shape == v.shape and k.stride() != v.stride()
    rows = torch.zeros(3, 128, dtype=torch.bfloat16)
    lens = torch.zeros(3, dtype=torch.int32)
    wide = torch.zeros(3, 4, dtype=torch.int32)
    one = torch.zeros(3, dtype=torch.int32).as_strided((3, 1), (1, 3))
    for pages in ((k, v), (v, k)):
        for table in (wide, one):
            with pytest.raises(ValueError, match="must be on a GPU"):
                ops.sdpa_decode_paged(rows, *pages, table, lens)
            with pytest.raises(ValueError, match="must be on a GPU"):
                ops.kv_append_paged(rows, rows, *pages, table, lens)
    other = torch.zeros(5, 2, 16, 128, dtype=torch.bfloat16)[:, :1]
    with pytest.raises(ValueError, match="v_pages must be as k_pages"):
        ops.sdpa_decode_paged(rows, k, other, wide, lens)
