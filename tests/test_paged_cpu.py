"""Batched attention serving without a GPU: the bounds that keep the kernels within their buffers
(nmi_paged.hpp compiled for the host), the launches' grids, refusals of the C ABI and of the torch
front end, and the oracle against independent forms."""
import ctypes
import math
import os
import random
import subprocess
import sys

import numpy as np
import pytest
import torch

from nemotron_infer_amd import _lib, build, ops
from oracle import attention, block, e4m3, linear, paged
from tests.test_host_runtime_cpu import host  # noqa: F401  (a fixture)

SHIM = """
#include "nmi_paged.hpp"
extern "C" {
int page(int id, int n, int* bad) { bool b = false; int r = nmi::checked_page(id, n, &b); *bad = b; return r; }
int len(int l, int max_pages, int shift, int* bad) {
    bool b = false; int r = nmi::checked_len(l, max_pages, shift, &b); *bad = b; return r;
}
int span(int c0, int c1, int tokens, int* first, int* bad) {
    bool b = false; int r = nmi::checked_span(c0, c1, tokens, first, &b); *bad = b; return r;
}
int share(unsigned total, int waves, int unit) { return nmi::range_tiles(total, waves, unit); }
unsigned first(unsigned x, int c, unsigned total) { return nmi::range_first(x, c, total); }
int joint(unsigned x, unsigned first, unsigned tiles, int c, unsigned total) { return nmi::is_joint(x, first, tiles, c, total); }
int pieces(unsigned first, unsigned tiles, int c, unsigned total, int* owners, int most) {
    const nmi::Pieces p = nmi::pieces_of(first, tiles, c, total);
    for (int i = 0; i < p.count() && i < most; ++i) owners[i] = p.owner(i);
    return p.count();
}
}
"""


@pytest.fixture(scope="module")
def bounds(tmp_path_factory):
    d = tmp_path_factory.mktemp("paged")
    src, so = d / "shim.cpp", str(d / "libshim.so")
    src.write_text(SHIM)
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-shared", "-fPIC", f"-I{build.CSRC}", str(src), "-o", so],
                   check=True, timeout=120)
    return ctypes.CDLL(so)


EDGES = [-2 ** 31, -2 ** 31 + 1, -7, -1, 0, 1, 2, 15, 16, 17, 100, 2 ** 30 - 1, 2 ** 30, 2 ** 31 - 1]


def test_a_page_id_never_leaves_the_pool(bounds):
    bad = ctypes.c_int()
    for n in (1, 2, 16, 2 ** 31 - 1):
        for i in EDGES:
            got = bounds.page(i, n, ctypes.byref(bad))
            assert 0 <= got < n
            assert bool(bad.value) == (not 0 <= i < n)
            assert bad.value or got == i


def test_a_length_never_leaves_its_row_of_the_table(bounds):
    bad = ctypes.c_int()
    for max_pages, shift in ((1, 4), (3, 4), (1, 20), (2 ** 26, 4), (2 ** 10, 20)):
        cap = max_pages << shift
        for n in EDGES + [cap - 1, cap, min(cap + 1, 2 ** 31 - 1)]:
            got = bounds.len(n, max_pages, shift, ctypes.byref(bad))
            assert got == max(0, min(n, cap)) and bool(bad.value) == (n > cap)


def test_a_packed_sequence_never_leaves_the_rows(bounds):
    bad, first = ctypes.c_int(), ctypes.c_int()
    for tokens in (1, 17, 2 ** 31 - 1):
        for c0 in EDGES:
            for c1 in EDGES:
                n = bounds.span(c0, c1, tokens, ctypes.byref(first), ctypes.byref(bad))
                assert n >= 0 and 0 <= first.value and first.value + n <= tokens
                good = 0 <= c0 <= c1 <= tokens
                assert bool(bad.value) == (not good)
                assert not good or (first.value, n) == (c0, c1 - c0)


def test_shares_cover_the_sequences_and_their_pieces_have_slots_of_their_own(bounds):
    """Whatever the lengths: the waves' shares are the whole row of tiles, each once; the pieces that the
    waves and workgroups make of a sequence are, in order, those that the joining kernel looks for; no
    two pieces share a slot, and every slot is in the workspace's waves + batch."""
    rng = random.Random(5)
    bounds.first.restype = ctypes.c_uint
    owners = (ctypes.c_int * 700)()
    joints = 0
    for trial in range(1500):
        batch, waves, unit = rng.randint(1, 60), 4 * rng.randint(1, 150), rng.choice([1, 2])
        top = int(math.exp(rng.uniform(0, math.log(2 ** 26 // batch))))
        tiles = [rng.choice([1, 1, top, rng.randint(1, top)]) for _ in range(batch)]
        if trial % 3 == 0:                               # ends of shares that are ends of sequences
            tiles = [rng.choice([1, 2, 4, 8, 16]) for _ in range(batch)]
        total = sum(tiles)
        c = bounds.share(total, waves, unit)
        assert c >= unit and waves * c >= total
        starts = [sum(tiles[:b]) for b in range(batch)]
        made = [[] for _ in range(batch)]
        slots = set()

        def piece(x, b, whole):
            assert x + b not in slots and x + b < waves + batch
            slots.add(x + b)
            made[b].append((x, whole))

        for x in range(waves // 4):                      # as the kernel goes through its share
            at, end = bounds.first(4 * x, c, total), bounds.first(4 * x + 4, c, total)
            if at >= end:
                continue
            b = max(i for i in range(batch) if starts[i] <= at)
            if bounds.joint(x, starts[b], tiles[b], c, total):
                assert end <= starts[b] + tiles[b]
                piece(4 * x, b, end - at == tiles[b])
                joints += 1
                continue
            for w in range(4 * x, 4 * x + 4):
                at, end = bounds.first(w, c, total), bounds.first(w + 1, c, total)
                assert end - at <= c
                while at < end:
                    b = max(i for i in range(batch) if starts[i] <= at)
                    stop = min(end, starts[b] + tiles[b])
                    piece(w, b, stop - at == tiles[b])
                    at = stop
        for b in range(batch):
            n = bounds.pieces(starts[b], tiles[b], c, total, owners, 700)
            assert [x for x, _ in made[b]] == owners[:n]
            assert (n == 1) == made[b][0][1]
    assert joints > 1000
    # as many tiles as a call may have
    c = bounds.share(2 ** 31 - 1, 4, 1)
    assert c == 2 ** 29 and bounds.first(3, c, 2 ** 31 - 1) == 3 * 2 ** 29
    assert bounds.first(4, c, 2 ** 31 - 1) == bounds.first(2 ** 24, c, 2 ** 31 - 1) == 2 ** 31 - 1


# --- the oracle ------------------------------------------------------------------------------------


def _bits(shape, seed, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * scale).to(torch.bfloat16).view(torch.int16).numpy().view(np.uint16)


def _f64(bits):
    return linear.bf16_to_f32(bits).astype(np.float64)


@pytest.mark.parametrize("H,n_kv,n", [(5, 1, 1), (8, 2, 33), (4, 4, 50)])
def test_oracle_decode_is_the_contiguous_one_over_scattered_pages(H, n_kv, n):
    page, q = 16, _bits((1, H, 128), 1)
    kp, vp = _bits((7, n_kv, page, 128), 2), _bits((7, n_kv, page, 128), 3)
    table = np.array([[5, 0, 6, 2]])
    kc, vc = (np.concatenate([p[i] for i in table[0]], axis=1) for p in (kp, vp))
    got = paged.decode(_f64(q), _f64(kp), _f64(vp), table, [n])
    assert np.allclose(got[0], attention.sdpa_decode_f64(q[0], kc, vc, n), rtol=1e-12, atol=1e-14)
    wrong = paged.decode(_f64(q), _f64(kp), _f64(vp), table[:, ::-1], [n])
    assert not np.allclose(wrong, got, rtol=1e-3)
    assert not paged.decode(_f64(q), _f64(kp), _f64(vp), table, [0]).any()


def test_oracle_prefill_is_each_prompt_alone():
    H, n_kv, cu = 4, 2, [2, 9, 9, 10, 30]
    q, k, v = _bits((32, H * 128), 4), _bits((32, n_kv * 128), 5), _bits((32, n_kv * 128), 6)
    got = paged.prefill(_f64(q).reshape(32, H, 128), _f64(k).reshape(32, n_kv, 128), _f64(v).reshape(32, n_kv, 128), cu)
    for a, b in zip(cu, cu[1:]):
        if b > a:
            want = attention.sdpa_prefill_f64(q[a:b], k[a:b], v[a:b], n_kv)
            assert np.allclose(got[a:b].reshape(b - a, -1), want, rtol=1e-12, atol=1e-14)
    assert np.isnan(got[:2]).all() and np.isnan(got[30:]).all()


@pytest.mark.parametrize("interleaved", [False, True])
def test_oracle_rotation(interleaved):
    x = _f64(_bits((3, 2, 128), 7))
    pos, f = np.array([0, 1, 100000]), 10000.0 ** (-np.arange(16) / 16)
    got = paged.rotate(x, pos, f, interleaved)
    assert np.array_equal(got[0], x[0]) and np.array_equal(got[..., 32:], x[..., 32:])
    pairs = (lambda y: y[..., 0:32:2] + 1j * y[..., 1:32:2]) if interleaved else (lambda y: y[..., :16] + 1j * y[..., 16:32])
    want = pairs(x) * np.exp(1j * pos[:, None] * f)[:, None]
    assert np.allclose(pairs(got), want, atol=1e-9)
    other = paged.rotate(x, pos, f, not interleaved)
    assert not np.allclose(other[1:], got[1:], atol=1e-2)


def test_oracle_e4m3_rounding_is_the_formats():
    lut = e4m3.decode_lut()[:0x7F].astype(np.float64)
    mid = (lut[1:] + lut[:-1]) / 2
    x = np.concatenate([lut, mid, np.nextafter(mid, 0), np.nextafter(mid, 1e9), [447.0, 500.0, 1e30]])
    x = np.concatenate([x, -x])
    want = e4m3.decode_lut()[e4m3.quantize_rne(np.clip(x, -448, 448).astype(np.float32))]
    near = np.clip(x, -448, 448).astype(np.float32).astype(np.float64) == np.clip(x, -448, 448)
    assert near.sum() > 300 and np.array_equal(paged.round_e4m3(x)[near], want[near])
    assert np.isnan(paged.round_e4m3(np.nan))


# --- launches --------------------------------------------------------------------------------------

CACHE = """
W, ST = 1 << 38, 1 << 12
def cache(kind=0, page=16, max_pages=64, n_kv=8):
    return _lib.PagedKv(W, W, n_kv * page * 128, page * 128, 128, W, max_pages, None, None, kind, 100, page, max_pages, n_kv)
def decode(batch, H, **kw):
    c = cache(**kw)
    need = L.nmi_sdpa_decode_paged_workspace_bytes(batch, H, c.n_kv_heads)
    rc = L.nmi_sdpa_decode_paged(ctypes.addressof(c), W, H * 128, W, H * 128, W, batch, H, 0.1, W, need, ST)
    assert rc == 0, L.nmi_last_error()
    return [need, [l[1:] for l in launches()]]
"""


def test_decode_launches_fit_the_workspace(host):  # noqa: F811
    """Two resident workgroups per CU (256 CUs) at most, and slots for their waves' pieces in the
    workspace, whatever the batch, the heads and the cache; the joining launch reaches every head of every
    sequence."""
    got = host(CACHE + """
result = [[b, h, n, kind, decode(b, h, n_kv=n, kind=kind)] for b in (1, 3, 8, 9, 64, 1000)
          for h, n in ((40, 8), (4, 4), (33, 1)) for kind in (0, 1)]
""")
    for b, h, n, kind, (need, grids) in got:
        (x, y, z, threads), (jx, jy, jz, jthreads) = grids
        assert need == (4 * x + b) * h * 130 * 4 + 16 * b and y == n and z == -(-(h // n) // 16) and threads == 256
        assert 512 - y * z < x * y * z <= 512
        assert jx == b and jy == -(-h // min(8, -(-b * h // 2048))) and jz == 1 and jthreads == 256


def test_packed_prefill_launches_enough_workgroups(host):  # noqa: F811
    """As many as `tokens` rows in `batch` sequences can need: of a sequence's last tile, one for each head
    (more than 64 rows, or a launch that is resident at once), two or four heads of a group (fewer rows)."""
    grids = host("""
W, ST = 1 << 38, 1 << 12
result = []
for H, n_kv in ((16, 4), (40, 8), (6, 2), (7, 1)):
    for tokens, batch in ((1, 1), (1, 50), (127, 3), (128, 1), (128, 2), (5000, 7), (300, 1000), (2000, 60), (2000, 30), (9000, 70)):
        rc = L.nmi_sdpa_prefill_packed_bf16(W, H * 128, W, n_kv * 128, W, n_kv * 128, W, H * 128, W, batch, tokens, H, n_kv, 0.1, ST)
        assert rc == 0, L.nmi_last_error()
        result.append([H, n_kv, tokens, batch, launches()[-1][1]])
""")
    for H, n_kv, tokens, batch, x in grids:
        n, group = min(batch, tokens), H // n_kv
        shared = (tokens // 128 + n) * H > 2 * 256

        def workgroups(v):
            rows = v - v // 128 * 128 or 128
            heads = 1 if rows > 64 or not shared else 2 if rows > 32 else 4
            return (-(-v // 128) - 1) * H + n_kv * -(-group // heads) if v else 0

        # n sequences, all of one row but the last; and as many as can be whose last tile just needs more
        tries = [[1] * (n - 1) + [tokens - n + 1]]
        for full in (0, 128, 256):
            for v in (full + 1, full + 33, full + 65):
                m = min(n, tokens // v)
                tries.append([v] * m + ([tokens - m * v] if m < n else []))
        assert x >= max(sum(workgroups(v) for v in lens) for lens in tries if lens), (H, tokens, batch)


# --- refusals --------------------------------------------------------------------------------------

FAKE = 0x10000


def _cache(**kw):
    c = _lib.PagedKv(FAKE, FAKE, 8 * 16 * 128, 16 * 128, 128, FAKE, 4, None, None, 0, 10, 16, 4, 8)
    for k, v in kw.items():
        setattr(c, k, v)
    return c


BAD_CACHES = [
    (dict(k_pages=0), _lib.NMI_ERR_INVALID_ARG), (dict(v_pages=0), _lib.NMI_ERR_INVALID_ARG),
    (dict(page_table=0), _lib.NMI_ERR_INVALID_ARG), (dict(kv_type=2), _lib.NMI_ERR_INVALID_ARG),
    (dict(page_size=8), _lib.NMI_ERR_INVALID_ARG), (dict(page_size=24), _lib.NMI_ERR_INVALID_ARG),
    (dict(page_size=0), _lib.NMI_ERR_INVALID_ARG), (dict(page_size=1 << 21), _lib.NMI_ERR_INVALID_ARG),
    (dict(page_size=-16), _lib.NMI_ERR_INVALID_ARG), (dict(n_pages=0), _lib.NMI_ERR_INVALID_ARG),
    (dict(max_pages=0), _lib.NMI_ERR_INVALID_ARG), (dict(max_pages=5), _lib.NMI_ERR_INVALID_ARG),
    (dict(max_pages=2 ** 26 + 1, page_table_stride=2 ** 27), _lib.NMI_ERR_INVALID_ARG),
    (dict(n_kv_heads=0), _lib.NMI_ERR_INVALID_ARG), (dict(token_stride=64), _lib.NMI_ERR_INVALID_ARG),
    (dict(token_stride=2 ** 24 + 8), _lib.NMI_ERR_INVALID_ARG), (dict(head_stride=-128), _lib.NMI_ERR_INVALID_ARG),
    (dict(page_stride=0), _lib.NMI_ERR_INVALID_ARG), (dict(k_scale=FAKE), _lib.NMI_ERR_INVALID_ARG),
    (dict(k_pages=FAKE + 8), _lib.NMI_ERR_ALIGNMENT), (dict(token_stride=132), _lib.NMI_ERR_ALIGNMENT),
    (dict(kv_type=1, token_stride=136), _lib.NMI_ERR_ALIGNMENT), (dict(page_table=FAKE + 2), _lib.NMI_ERR_ALIGNMENT),
    (dict(kv_type=1, v_scale=FAKE + 1), _lib.NMI_ERR_ALIGNMENT),
]


def _append(c, q=FAKE, ldq=5120, k=FAKE, ldk=1024, v=FAKE, ldv=1024, qo=FAKE, ldqo=5120, ko=FAKE, ldko=1024, cu=FAKE,
            start=FAKE, batch=2, tokens=9, H=40, inv=FAKE, rotary=64):
    return _lib.lib().nmi_kv_append_paged(ctypes.addressof(c) if c else None, q, ldq, k, ldk, v, ldv, qo, ldqo, ko, ldko,
                                          cu, start, batch, tokens, H, inv, rotary, 0, None)


def _decode(c, q=FAKE, ldq=5120, o=FAKE, ldo=5120, lens=FAKE, batch=2, H=40, scale=0.1, ws=FAKE, ws_bytes=1 << 30):
    return _lib.lib().nmi_sdpa_decode_paged(ctypes.addressof(c) if c else None, q, ldq, o, ldo, lens, batch, H, scale, ws,
                                            ws_bytes, None)


@pytest.mark.parametrize("change,code", BAD_CACHES)
def test_bad_caches_are_refused(change, code):
    L = _lib.lib()
    assert _append(_cache(**change)) == code and L.nmi_last_error().decode().startswith("nmi_kv_append_paged")
    assert _decode(_cache(**change)) == code and L.nmi_last_error().decode().startswith("nmi_sdpa_decode_paged")


@pytest.mark.parametrize("change,code", [
    (dict(k=0), _lib.NMI_ERR_INVALID_ARG), (dict(v=0), _lib.NMI_ERR_INVALID_ARG), (dict(start=0), _lib.NMI_ERR_INVALID_ARG),
    (dict(batch=0), _lib.NMI_ERR_INVALID_ARG), (dict(tokens=0), _lib.NMI_ERR_INVALID_ARG),
    (dict(cu=0), _lib.NMI_ERR_INVALID_ARG),                                  # 9 tokens of 2 sequences
    (dict(rotary=-16), _lib.NMI_ERR_INVALID_ARG), (dict(rotary=72), _lib.NMI_ERR_INVALID_ARG),
    (dict(rotary=144), _lib.NMI_ERR_INVALID_ARG), (dict(rotary=0), _lib.NMI_ERR_INVALID_ARG),
    (dict(inv=0), _lib.NMI_ERR_INVALID_ARG), (dict(q=0), _lib.NMI_ERR_INVALID_ARG), (dict(qo=0), _lib.NMI_ERR_INVALID_ARG),
    (dict(q=0, qo=0, rotary=0, inv=0), _lib.NMI_ERR_INVALID_ARG),           # k_out without a rotation
    (dict(H=41), _lib.NMI_ERR_INVALID_ARG), (dict(H=0), _lib.NMI_ERR_INVALID_ARG),
    (dict(k=FAKE + 8), _lib.NMI_ERR_ALIGNMENT), (dict(ldk=1020), _lib.NMI_ERR_ALIGNMENT),
    (dict(ldv=1028), _lib.NMI_ERR_ALIGNMENT), (dict(ldq=5112), _lib.NMI_ERR_ALIGNMENT),
    (dict(ldqo=2 ** 24 + 8), _lib.NMI_ERR_ALIGNMENT), (dict(ko=FAKE + 4), _lib.NMI_ERR_ALIGNMENT),
    (dict(cu=FAKE + 1), _lib.NMI_ERR_ALIGNMENT), (dict(inv=FAKE + 2), _lib.NMI_ERR_ALIGNMENT),
])
def test_append_refuses(change, code):
    assert _append(_cache(), **change) == code
    assert _append(None) == _lib.NMI_ERR_INVALID_ARG


@pytest.mark.parametrize("change,code", [
    (dict(q=0), _lib.NMI_ERR_INVALID_ARG), (dict(o=0), _lib.NMI_ERR_INVALID_ARG), (dict(lens=0), _lib.NMI_ERR_INVALID_ARG),
    (dict(batch=0), _lib.NMI_ERR_INVALID_ARG), (dict(H=4), _lib.NMI_ERR_INVALID_ARG), (dict(H=41), _lib.NMI_ERR_INVALID_ARG),
    (dict(scale=0.0), _lib.NMI_ERR_INVALID_ARG), (dict(scale=-1.0), _lib.NMI_ERR_INVALID_ARG),
    (dict(scale=math.inf), _lib.NMI_ERR_INVALID_ARG), (dict(scale=math.nan), _lib.NMI_ERR_INVALID_ARG),
    (dict(q=FAKE + 2), _lib.NMI_ERR_ALIGNMENT), (dict(ldq=5121), _lib.NMI_ERR_ALIGNMENT),
    (dict(ldo=5119), _lib.NMI_ERR_ALIGNMENT), (dict(o=FAKE + 2), _lib.NMI_ERR_ALIGNMENT),
    (dict(lens=FAKE + 2), _lib.NMI_ERR_ALIGNMENT), (dict(ws=FAKE + 8), _lib.NMI_ERR_ALIGNMENT),
    (dict(ws_bytes=1000), _lib.NMI_ERR_WORKSPACE),
])
def test_decode_refuses(change, code):
    assert _decode(_cache(), **change) == code
    assert _decode(None) == _lib.NMI_ERR_INVALID_ARG


def test_decode_refuses_more_positions_than_it_can_count():
    assert _decode(_cache(max_pages=2 ** 26, page_table_stride=2 ** 26), batch=32) == _lib.NMI_ERR_INVALID_ARG
    assert _lib.lib().nmi_sdpa_decode_paged_workspace_bytes(0, 40, 8) == 0
    assert _lib.lib().nmi_sdpa_decode_paged_workspace_bytes(1, 41, 8) == 0


@pytest.mark.parametrize("change,code", [
    (dict(q=0), _lib.NMI_ERR_INVALID_ARG), (dict(cu=0), _lib.NMI_ERR_INVALID_ARG), (dict(batch=0), _lib.NMI_ERR_INVALID_ARG),
    (dict(tokens=0), _lib.NMI_ERR_INVALID_ARG), (dict(H=41), _lib.NMI_ERR_INVALID_ARG),
    (dict(n_kv=0), _lib.NMI_ERR_INVALID_ARG), (dict(scale=0.0), _lib.NMI_ERR_INVALID_ARG),
    (dict(scale=math.nan), _lib.NMI_ERR_INVALID_ARG), (dict(tokens=2 ** 31 - 1, batch=2 ** 31 - 1), _lib.NMI_ERR_INVALID_ARG),
    (dict(q=FAKE + 8), _lib.NMI_ERR_ALIGNMENT), (dict(ldk=1016), _lib.NMI_ERR_ALIGNMENT),
    (dict(ldv=1028), _lib.NMI_ERR_ALIGNMENT), (dict(ldk=2 ** 24 + 8), _lib.NMI_ERR_ALIGNMENT),
    (dict(ldo=5122), _lib.NMI_ERR_ALIGNMENT), (dict(o=FAKE + 4), _lib.NMI_ERR_ALIGNMENT),
    (dict(cu=FAKE + 2), _lib.NMI_ERR_ALIGNMENT),
])
def test_packed_prefill_refuses(change, code):
    a = dict(q=FAKE, ldq=5120, k=FAKE, ldk=1024, v=FAKE, ldv=1024, o=FAKE, ldo=5120, cu=FAKE, batch=2, tokens=9, H=40, n_kv=8,
             scale=0.1)
    a.update(change)
    assert _lib.lib().nmi_sdpa_prefill_packed_bf16(*a.values(), None) == code


def _tensors(T=3, n_kv=2, H=4, kind=torch.bfloat16):
    z = lambda *s: torch.zeros(*s, dtype=torch.bfloat16)  # noqa: E731
    ints = lambda n: torch.zeros(n, dtype=torch.int32)  # noqa: E731
    pages = torch.zeros(5, n_kv, 16, 128).to(kind)
    return dict(q=z(T, H * 128), k=z(T, n_kv * 128), v=z(T, n_kv * 128), k_pages=pages, v_pages=pages.clone(),
                page_table=torch.zeros(T, 4, dtype=torch.int32), start_pos=ints(T), kv_lens=ints(T),
                inv_freq=torch.ones(32))


def test_valid_cpu_calls_are_refused_before_the_library():
    t = _tensors()
    with pytest.raises(ValueError, match="GPU"):
        ops.kv_append_paged(t["k"], t["v"], t["k_pages"], t["v_pages"], t["page_table"], t["start_pos"], q=t["q"],
                            inv_freq=t["inv_freq"])
    with pytest.raises(ValueError, match="GPU"):
        ops.sdpa_decode_paged(t["q"], t["k_pages"], t["v_pages"], t["page_table"], t["kv_lens"])
    with pytest.raises(ValueError, match="GPU"):
        ops.sdpa_prefill_packed_bf16(t["q"], t["k"], t["v"], torch.zeros(2, dtype=torch.int32), 4, 2)


@pytest.mark.parametrize("name,value,exc", [
    ("k_pages", torch.zeros(5, 2, 16, 64, dtype=torch.bfloat16), ValueError),
    ("k_pages", torch.zeros(5, 2, 16, 128, dtype=torch.float16), TypeError),
    ("v_pages", torch.zeros(5, 2, 16, 128, dtype=torch.uint8), ValueError),
    ("v_pages", torch.zeros(5, 16, 2, 128, dtype=torch.bfloat16).transpose(1, 2), ValueError),     # other strides
    ("k_pages", torch.zeros(5, 2, 128, 16, dtype=torch.bfloat16).transpose(2, 3), ValueError),
    ("page_table", torch.zeros(3, 4, dtype=torch.int64), ValueError),
    ("page_table", torch.zeros(2, 4, dtype=torch.int32), ValueError),
    ("page_table", torch.zeros(4, 3, dtype=torch.int32).t()[:, ::2], ValueError),
])
def test_front_end_refuses_bad_caches(name, value, exc):
    t = _tensors()
    t[name] = value
    for call in (lambda: ops.sdpa_decode_paged(t["q"], t["k_pages"], t["v_pages"], t["page_table"], t["kv_lens"]),
                 lambda: ops.kv_append_paged(t["k"], t["v"], t["k_pages"], t["v_pages"], t["page_table"], t["start_pos"])):
        with pytest.raises(exc) as e:
            call()
        assert "on a GPU" not in str(e.value)       # (the last check, which these tensors would fail)


def test_front_end_refuses_bad_operands():
    t = _tensors()
    cache = (t["k_pages"], t["v_pages"], t["page_table"])
    scale = torch.ones(2)
    for call in (
            lambda: ops.sdpa_decode_paged(t["q"][:, :384], *cache, t["kv_lens"]),             # 3 heads for 2
            lambda: ops.sdpa_decode_paged(t["q"].float(), *cache, t["kv_lens"]),
            lambda: ops.sdpa_decode_paged(t["q"], *cache, t["kv_lens"].long()),
            lambda: ops.sdpa_decode_paged(t["q"], *cache, t["kv_lens"][:2]),
            lambda: ops.sdpa_decode_paged(t["q"], *cache, t["kv_lens"], k_scale=scale),       # bf16 cache
            lambda: ops.sdpa_decode_paged(t["q"], *cache, t["kv_lens"], out=t["q"][:2]),
            lambda: ops.kv_append_paged(t["k"][:2], t["v"][:2], *cache, t["start_pos"]),      # 2 rows, 3 sequences
            lambda: ops.kv_append_paged(t["k"], t["v"][:2], *cache, t["start_pos"]),
            lambda: ops.kv_append_paged(t["k"], t["v"], *cache, t["start_pos"].long()),
            lambda: ops.kv_append_paged(t["k"], t["v"], *cache, t["start_pos"], q=t["q"]),    # no rotation
            lambda: ops.kv_append_paged(t["k"], t["v"], *cache, t["start_pos"], k_out=t["k"]),
            lambda: ops.kv_append_paged(t["k"], t["v"], *cache, t["start_pos"], inv_freq=t["inv_freq"].double()),
            lambda: ops.kv_append_paged(t["k"], t["v"], *cache, t["start_pos"], inv_freq=t["inv_freq"], q_out=t["q"]),
            lambda: ops.kv_append_paged(t["k"], t["v"], *cache, t["start_pos"], cu_seqlens=t["start_pos"]),
            lambda: ops.sdpa_prefill_packed_bf16(t["q"], t["k"], t["v"], torch.zeros(2), 4, 2),
            lambda: ops.sdpa_prefill_packed_bf16(t["q"], t["k"][:2], t["v"], torch.zeros(2, dtype=torch.int32), 4, 2),
            lambda: ops.sdpa_prefill_packed_bf16(t["q"], t["k"], t["v"], torch.zeros(0, dtype=torch.int32), 4, 2)):
        with pytest.raises(ValueError) as e:
            call()
        assert "on a GPU" not in str(e.value)
    e = _tensors(kind=torch.float8_e4m3fn)
    with pytest.raises(ValueError, match="k_scale"):
        ops.sdpa_decode_paged(e["q"], e["k_pages"], e["v_pages"], e["page_table"], e["kv_lens"], k_scale=torch.ones(3))


def test_block_rounding_helper_is_nearest_even():
    assert np.array_equal(_f64(block.bf16_round_exact(np.array([1.0, 1 + 2.0 ** -8, 1 + 3 * 2.0 ** -8]))),
                          [1.0, 1.0, 1 + 2.0 ** -6])


def test_front_end_errors_are_exceptions_and_keep_no_references():
    """Arguments of any kind end in a Python exception, never past it; what was passed is let go."""
    t = _tensors()
    cache = (t["k_pages"], t["v_pages"], t["page_table"])
    odd = [None, 3, "x", object(), torch.zeros(2, 2).to_sparse(), torch.empty(3, 256, dtype=torch.bfloat16, device="meta"),
           torch.zeros(()), torch.zeros(0)]
    calls = [
        lambda x: ops.sdpa_decode_paged(t["q"], x, t["v_pages"], t["page_table"], t["kv_lens"]),
        lambda x: ops.sdpa_decode_paged(t["q"], t["k_pages"], x, t["page_table"], t["kv_lens"]),
        lambda x: ops.sdpa_decode_paged(t["q"], t["k_pages"], t["v_pages"], x, t["kv_lens"]),
        lambda x: ops.sdpa_decode_paged(t["q"], *cache, x),
        lambda x: ops.sdpa_decode_paged(x, *cache, t["kv_lens"]),
        lambda x: ops.sdpa_decode_paged(t["q"], *cache, t["kv_lens"], out=x),
        lambda x: ops.sdpa_decode_paged(t["q"], *cache, t["kv_lens"], scale=x),
        lambda x: ops.kv_append_paged(x, t["v"], *cache, t["start_pos"]),
        lambda x: ops.kv_append_paged(t["k"], x, *cache, t["start_pos"]),
        lambda x: ops.kv_append_paged(t["k"], t["v"], *cache, x),
        lambda x: ops.kv_append_paged(t["k"], t["v"], *cache, t["start_pos"], cu_seqlens=x),
        lambda x: ops.kv_append_paged(t["k"], t["v"], *cache, t["start_pos"], q=x, inv_freq=t["inv_freq"]),
        lambda x: ops.kv_append_paged(t["k"], t["v"], *cache, t["start_pos"], q=t["q"], inv_freq=x),
        lambda x: ops.sdpa_prefill_packed_bf16(x, t["k"], t["v"], t["start_pos"], 4, 2),
        lambda x: ops.sdpa_prefill_packed_bf16(t["q"], t["k"], t["v"], x, 4, 2),
        lambda x: ops.sdpa_prefill_packed_bf16(t["q"], t["k"], t["v"], t["start_pos"], x, 2),
    ]
    held = [*odd[3:], *t.values()]
    before = [sys.getrefcount(x) for x in held]
    for _ in range(3):
        for call in calls:
            for x in odd:
                with pytest.raises((ValueError, TypeError, RuntimeError, AttributeError)):
                    call(x)
    del call, x
    assert [sys.getrefcount(x) for x in held] == before
    pages = torch.zeros(4, 0, 16, 128, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="no KV heads"):
        ops.sdpa_decode_paged(t["q"], pages, pages, t["page_table"], t["kv_lens"])
    from nemotron_infer_amd.csrc import front
    for f in (front.kv_append_paged, front.sdpa_decode_paged, front.sdpa_prefill_packed_bf16):
        with pytest.raises(TypeError, match="expected"):
            f(1, 2)

