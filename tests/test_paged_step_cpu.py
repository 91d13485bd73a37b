"""The life of a serving step on a paged cache without a GPU: the arithmetic behind block scales, packed pieces and
grids (nmi_paged.hpp compiled for the host), the launches, refusals of the C ABI and of the torch front end, and the
oracle against independent forms."""
import ctypes
import math
import random
import subprocess
from fractions import Fraction

import numpy as np
import pytest
import torch

from nemotron_infer_amd import _lib, build, ops
from oracle import e4m3, paged
from tests.test_host_runtime_cpu import host  # noqa: F401  (a fixture)

SHIM = """
#include "nmi_paged.hpp"
extern "C" {
int exponent(unsigned b) { return nmi::block_exponent(b); }
int exponent_of_scale(unsigned b) { return nmi::block_exponent_of_scale(b); }
long long block(long long page, int n_kv, int head, int shift, int pos) { return nmi::block_index(page, n_kv, head, shift, pos); }
int span(int c0, int c1, int tokens, int before, int* first, int* place, int* bad) {
    bool b = false; int r = nmi::later_span(c0, c1, tokens, before, first, place, &b); *bad = b; return r;
}
int blocks(long long pos, int n) { return nmi::blocks_of(pos, n); }
long long most(long long tokens, long long batch) { return nmi::most_blocks(tokens, batch); }
int completed(long long pos, int n, int shift) { return nmi::pages_completed(pos, n, shift); }
long long most_completed(long long tokens, long long batch, int shift) { return nmi::most_pages_completed(tokens, batch, shift); }
}
"""
LL = ctypes.c_longlong


@pytest.fixture(scope="module")
def hpp(tmp_path_factory):
    d = tmp_path_factory.mktemp("step")
    src, so = d / "shim.cpp", str(d / "libshim.so")
    src.write_text(SHIM)
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-shared", "-fPIC", f"-I{build.CSRC}", str(src), "-o", so],
                   check=True, timeout=120)
    so = ctypes.CDLL(so)
    so.block.restype = so.most.restype = so.most_completed.restype = LL
    return so


def _bits(x):
    return int(np.float32(x).view(np.uint32))


def _scale(e):
    return Fraction(2) ** (e - 127)


def test_a_blocks_scale_is_the_smallest_power_of_two_that_holds_it(hpp):
    """Around every border 448 * 2^e = 1.75 * 2^(e + 8), at the ends of float32, and at random."""
    rng = np.random.default_rng(1)
    tries = [0, 1, 0x7FFFFF, 0x800000, 0x7F7FFFFF]
    for e in range(1, 255):
        tries += [e << 23, (e << 23) + 1, (e << 23) | 0x5FFFFF, (e << 23) | 0x600000, (e << 23) | 0x600001, (e << 23) | 0x7FFFFF]
    tries += [int(b) for b in rng.integers(0, 0x7F800000, 3000)]
    for b in tries:
        amax, e = Fraction(float(np.uint32(b).view(np.float32))), hpp.exponent(ctypes.c_uint(b))
        assert 1 <= e <= 247 and amax <= 448 * _scale(e), hex(b)
        assert e == 1 or amax > 448 * _scale(e - 1), hex(b)
        assert float(_scale(e)) == paged.block_scale(float(amax))


def test_a_scale_found_in_memory_is_raised_to_a_power_of_two(hpp):
    for x in (2.0 ** -126, 2.0 ** -30, 0.5, 1.0, 3.0, 0.01, 1.5 * 2.0 ** 100, 2.0 ** 120, 1e-40):
        e = hpp.exponent_of_scale(ctypes.c_uint(_bits(x)))
        s = float(_scale(e))
        assert s >= np.float32(x) and (s / 2 < np.float32(x) or e == 1)
    for b in (0, 0x80000000, _bits(np.inf), _bits(np.nan), 0xFFFFFFFF, _bits(-1.0), 0xFF7FFFFF):     # no scales
        assert hpp.exponent_of_scale(ctypes.c_uint(b)) == 1
    assert hpp.exponent_of_scale(ctypes.c_uint(0x7F7FFFFF)) == 253                 # (of which there is an inverse)


def test_a_positions_scale_is_its_blocks(hpp):
    for shift in (4, 5, 8, 20):
        size = 1 << shift
        for page, n_kv, head in ((0, 1, 0), (3, 8, 5), (2 ** 31 - 1, 65535, 65534)):
            for pos in (0, 15, 16, size - 1, size, 5 * size + 17 % size, 2 ** 30 - 1):
                want = (page * n_kv + head) * (size // 16) + pos % size // 16
                assert hpp.block(LL(page), n_kv, head, shift, pos) == want


def _span(hpp, c0, c1, tokens, before):
    first, place, bad = ctypes.c_int(), ctypes.c_int(), ctypes.c_int()
    n = hpp.span(c0, c1, tokens, before, ctypes.byref(first), ctypes.byref(place), ctypes.byref(bad))
    return n, first.value, place.value, bool(bad.value)


def test_no_row_is_two_sequences(hpp):
    """Whatever the offsets: the sequences' rows are within those given, none twice, at their places; offsets in
    order give every row, and nothing is reported."""
    rng = random.Random(2)
    for trial in range(3000):
        tokens, batch = rng.randint(1, 60), rng.randint(1, 12)
        if trial % 2:
            cu = sorted(rng.randint(0, tokens) for _ in range(batch + 1))
        else:
            cu = [rng.choice([rng.randint(-5, tokens + 5), -2 ** 31, 2 ** 31 - 1, 0, tokens]) for _ in range(batch + 1)]
        end, seen = 0, set()
        for c0, c1 in zip(cu, cu[1:]):
            n, first, place, bad = _span(hpp, c0, c1, tokens, end)
            assert n >= 0 and place >= 0
            rows = set(range(first, first + n))
            assert not rows & seen and all(0 <= r < tokens for r in rows)
            if trial % 2:
                assert not bad and (n, place) == (c1 - c0, 0) and (not n or first == c0)
            elif n:
                assert place == first - max(c0, 0) and first + n == min(c1, tokens)
            seen |= rows
            whole = max(0, min(c1, tokens) - min(max(c0, 0), tokens)) if c1 > c0 else 0
            assert bad or whole == n
            end = max(end, min(c1, tokens) if whole else 0)
        assert not trial % 2 or seen == set(range(cu[0], cu[-1]))


def test_grids_hold_every_block_and_page(hpp):
    """As many workgroups as the rows can need, whatever the positions; and the counts themselves."""
    rng = random.Random(3)
    for trial in range(4000):
        batch = rng.randint(1, 40)
        if trial % 2:
            lens = [rng.choice([0, 1, 2, 3, 16, 17, 18, 33, 34, rng.randint(0, 300)]) for _ in range(batch)]
            starts = [rng.choice([15, 15, 0, rng.randint(0, 2 ** 30)]) for _ in range(batch)]
        else:                                            # the most blocks that rows can need
            n = rng.choice([2, 18, 34])
            lens, starts = [n] * batch, [15] * batch
        tokens = sum(lens)
        if not tokens:
            continue
        shift = rng.choice([4, 5, 8])
        blocks = pages = 0
        for s, n in zip(starts, lens):
            touched = len({p // 16 for p in range(s, s + n)})
            assert hpp.blocks(LL(s), n) == touched
            whole = sum((p + 1) % (1 << shift) == 0 for p in range(s, s + n))
            assert hpp.completed(LL(s), n, shift) == whole
            blocks, pages = blocks + touched, pages + whole
        assert blocks <= hpp.most(LL(tokens), LL(batch)) <= tokens
        assert pages <= hpp.most_completed(LL(tokens), LL(batch), shift)


# --- the oracle ------------------------------------------------------------------------------------


def test_oracle_pages_have_one_owner_each():
    """Many steps of random requests: every page is free or in one place of one sequence, none is lost; slots name the
    places; what is not granted changes nothing."""
    rng = random.Random(4)
    denied = ended = 0
    for trial in range(60):
        batch, page, n_pages, width = rng.randint(1, 9), 16, rng.randint(1, 30), rng.randint(1, 6)
        lens, table = [rng.choice([-1, 0]) for _ in range(batch)], [[-1] * width for _ in range(batch)]
        free, count = list(range(n_pages)), n_pages
        rng.shuffle(free)
        for _ in range(40):
            new = [rng.choice([-1, 0, 1, 1, 1, 5, 16, 40]) for _ in range(batch)]
            was = [list(r) for r in table]
            got = paged.assign(lens, new, table, free, count, page, True)
            for b in range(batch):
                assert got["start_pos"][b] in (-1, lens[b])
                if got["start_pos"][b] < 0:
                    assert table[b] == was[b] and got["kv_lens"][b] == 0
                    denied += new[b] > 0 and lens[b] >= 0
                ended += got["lens"][b] < lens[b]
                rows = got["slots"][got["cu_seqlens"][b]:got["cu_seqlens"][b + 1]]
                if got["start_pos"][b] < 0:
                    assert rows == [-1] * max(0, new[b])
                else:
                    assert rows == [table[b][p // page] * page + p % page for p in range(lens[b], lens[b] + new[b])]
            lens, count = got["lens"], got["free_count"][0]
            held = [table[b][i] for b in range(batch) for i in range(-(-max(0, lens[b]) // page))]
            assert sorted(held + free[:count]) == list(range(n_pages))
            lens = [0 if n < 0 and rng.random() < 0.5 else n for n in lens]
    assert denied > 100 and ended > 100


def test_oracle_blocks_filled_by_token_or_at_once_are_alike():
    """The same scale; codes alike but for those that were subnormal on the way."""
    rng = np.random.default_rng(5)
    x = rng.standard_normal((16, 2, 128)) * np.exp2(rng.integers(-3, 4, (16, 1, 1)))
    values, scales = np.zeros((2, 2, 16, 128)), np.full((2, 2, 1), np.nan)
    paged.append_blocks(values, scales, x, [(t, 0, t) for t in range(16)], [[0]], 16)
    for t in range(16):
        paged.append_blocks(values, scales, x, [(t, 0, t)], [[1]], 16)
    assert np.array_equal(scales[0], scales[1])
    assert np.array_equal(scales[0, :, 0], [paged.block_scale(np.abs(x[:, h]).max()) for h in range(2)])
    normal = np.abs(values[0]) >= 2.0 ** -6
    assert normal.mean() > 0.9 and np.array_equal(values[1][normal], values[0][normal])
    assert np.abs(values[1] - values[0]).max() <= 2.0 ** -9
    assert np.array_equal(paged.round_e4m3(values[0]), values[0])


def test_oracle_selection_bounds_every_key():
    rng = np.random.default_rng(6)
    k = rng.standard_normal((9, 2, 16, 128))
    q, table = rng.standard_normal((6, 128)), [3, 8, 0, 5, 1, 7, 2]
    bounds = paged.page_bounds(k)
    for h in range(6):
        top = (k[:, h // 3] @ q[h]).max(-1)
        assert (np.where(q[h] > 0, bounds[:, h // 3, 1], bounds[:, h // 3, 0]) @ q[h] >= top - 1e-9).all()
    kept = paged.select(q, bounds, table, 100, 16, 3)
    assert all(len(k) == 3 and k[-1] == 6 and k == sorted(k) for k in kept)
    assert paged.select(q, bounds, table, 48, 16, 3) == [[0, 1, 2]] * 2 and paged.select(q, bounds, table, 100, 16, 1) == [[6]] * 2
    same = np.repeat(bounds[:1], 9, axis=0)
    assert paged.select(q, same, table, 100, 16, 3) == [[0, 1, 6]] * 2             # ties: the earliest
    same[5, 1, 0, 7] = np.nan                                                      # page 5 is place 3
    assert paged.select(q, same, table, 100, 16, 2) == [[0, 6], [3, 6]]
    v = rng.standard_normal(k.shape)
    whole = paged.decode(q[None], k, v, [table], [100])
    assert np.allclose(paged.decode_selected(q[None], k, v, [table], [100], [[list(range(7))] * 2]), whole)
    assert not np.allclose(paged.decode_selected(q[None], k, v, [table], [100], [kept]), whole, rtol=1e-2)


# --- launches --------------------------------------------------------------------------------------

CACHE = """
W, ST = 1 << 38, 1 << 12
def cache(kind=2, page=16, max_pages=64, n_kv=8):
    s = None if kind == 0 else W
    return _lib.PagedKv(W, W, n_kv * page * 128, page * 128, 128, W, max_pages, s, s, kind, 100, page, max_pages, n_kv)
"""


def test_append_launches(host):  # noqa: F811
    got = host(CACHE + """
result = []
for tokens, batch, packed in ((1, 1, 0), (24, 24, 0), (9000, 9000, 0), (1, 1, 1), (8191, 1, 1), (300, 40, 1), (70, 500, 1)):
    for rotary in (0, 64):
        c = cache()
        rc = L.nmi_kv_append_paged(ctypes.addressof(c), W if rotary else None, 5120, W, 1024, W, 1024, W if rotary else None, 5120,
                                   None, 0, W if packed else None, W, batch, tokens, 40, W if rotary else None, rotary, 0, ST)
        assert rc == 0, L.nmi_last_error()
        result.append([tokens, batch, packed, [l[1:] for l in launches()]])
""")
    for tokens, batch, packed, launches in got:
        assert len(launches) == 1
        x, y, z, threads = launches[0]
        if packed:
            n = min(batch, tokens)
            assert x == min(tokens, (tokens + 30 * n) // 16) + 1 and y >= 1
        else:
            assert 4 * x >= tokens and y == 1
        assert z == 1 and threads == 256


def test_sparse_launches_fit_the_workspace(host):  # noqa: F811
    """Scores, the chosen pages, their lengths and the decode's own workspace, in turn; two launches less where there is
    nothing to choose, one less where few positions are attended."""
    got = host(CACHE + """
result = []
for batch, H, n_kv, kind, max_pages, select in ((1, 40, 8, 2, 1563, 32), (20, 32, 8, 0, 900, 63), (70, 4, 2, 1, 8, 1), (3, 16, 4, 2, 8, 8),
                                                (3, 16, 4, 2, 8, 2 ** 31 - 1)):
    c = cache(kind=kind, max_pages=max_pages, n_kv=n_kv)
    need = L.nmi_sdpa_decode_paged_sparse_workspace_bytes(batch, H, n_kv, max_pages, select)
    dense = L.nmi_sdpa_decode_paged_workspace_bytes(batch, H, n_kv)
    def call(n, sel=None):
        return L.nmi_sdpa_decode_paged_sparse(ctypes.addressof(c), W, H * 128, W, H * 128, W, W, select, sel, batch, H, 0.1, W, n, ST)
    assert call(need) == 0, L.nmi_last_error()
    first = [l[1:] for l in launches()]
    assert call(need, W) == 0 and call(need - 1) == _lib.NMI_ERR_WORKSPACE
    result.append([batch, H, n_kv, max_pages, select, need, dense, first, len(launches())])
""")
    for batch, H, n_kv, max_pages, select, need, dense, first, again in got:
        groups, up = batch * n_kv, lambda n: -(-n // 16) * 16
        decode = 1 if 16 * min(select, max_pages) <= 640 else 2
        if select >= max_pages:
            assert need == dense and len(first) == decode and again == decode + 1
            continue
        assert need == up(4 * groups * max_pages) + up(4 * groups * select) + up(4 * batch) + dense
        assert len(first) == again == 2 + decode
        assert first[0][0] % groups == 0 and first[0][0] // groups <= -(-max_pages // 16) and first[1][0] == groups
    assert {len(first) for *_, first, _ in got} == {1, 3, 4}


def test_decode_launches(host):  # noqa: F811
    """Under scales of blocks one launch, a workgroup to a sequence's KV head (and 16 of its heads), where the rows of the
    table hold few positions; two otherwise, and always over the older caches."""
    got = host(CACHE + """
result = []
for kind in (0, 1, 2):
    for batch, H, n_kv, page, max_pages in ((1, 40, 8, 16, 1), (1, 40, 8, 16, 40), (1, 40, 8, 16, 41), (31, 40, 8, 64, 16), (32, 40, 8, 64, 16),
                                            (300, 40, 8, 64, 17), (300, 33, 1, 32, 20)):
        c = cache(kind=kind, page=page, max_pages=max_pages, n_kv=n_kv)
        need = L.nmi_sdpa_decode_paged_workspace_bytes(batch, H, n_kv)
        rc = L.nmi_sdpa_decode_paged(ctypes.addressof(c), W, H * 128, W, H * 128, W, batch, H, 0.1, W, need, ST)
        assert rc == 0, L.nmi_last_error()
        result.append([kind, batch, H, n_kv, page * max_pages, [l[1:] for l in launches()]])
""")
    for kind, batch, H, n_kv, most, launches in got:
        z = -(-(H // n_kv) // 16)
        if kind == 2 and (most <= 640 or (most <= 1024 and batch * n_kv * z >= 256)):
            assert launches == [[batch, n_kv, z, 256]]
        else:
            assert len(launches) == 2 and launches[0][1:] == [n_kv, z, 256]


# --- refusals --------------------------------------------------------------------------------------

FAKE = 0x10000
BAD, ALIGN = _lib.NMI_ERR_INVALID_ARG, _lib.NMI_ERR_ALIGNMENT


def _cache(**kw):
    c = _lib.PagedKv(FAKE, FAKE, 8 * 16 * 128, 16 * 128, 128, FAKE, 4, FAKE, FAKE, 2, 10, 16, 4, 8)
    for k, v in kw.items():
        setattr(c, k, v)
    return c


def _append(c, tokens=9, batch=2):
    return _lib.lib().nmi_kv_append_paged(ctypes.addressof(c), None, 0, FAKE, 1024, FAKE, 1024, None, 0, None, 0, FAKE, FAKE, batch,
                                          tokens, 0, None, 0, 0, None)


def _sparse(c, q=FAKE, ldq=5120, o=FAKE, ldo=5120, lens=FAKE, bounds=FAKE, select=2, selected=FAKE, batch=2, H=40, scale=0.1,
            ws=FAKE, ws_bytes=1 << 30):
    return _lib.lib().nmi_sdpa_decode_paged_sparse(ctypes.addressof(c) if c else None, q, ldq, o, ldo, lens, bounds, select,
                                                   selected, batch, H, scale, ws, ws_bytes, None)


def _bounds(c, bounds=FAKE, cu=FAKE, start=FAKE, batch=2, tokens=9):
    return _lib.lib().nmi_kv_bounds_paged(ctypes.addressof(c) if c else None, bounds, cu, start, batch, tokens, None)


def _assign(**kw):
    a = dict(lens=FAKE, new=FAKE, table=FAKE, stride=4, max_pages=4, page=16, free=FAKE, count=FAKE, n_pages=10, batch=2, tokens=9,
             start=FAKE, kv=FAKE, cu=FAKE, slots=FAKE, lens_out=FAKE, count_out=FAKE)
    a.update(kw)
    return _lib.lib().nmi_kv_assign_paged(*a.values(), None)


@pytest.mark.parametrize("change,code", [
    (dict(k_scale=None), BAD), (dict(v_scale=None), BAD), (dict(kv_type=3), BAD), (dict(kv_type=-1), BAD), (dict(kv_type=0), BAD),
    (dict(k_scale=FAKE + 2), ALIGN), (dict(token_stride=136), ALIGN), (dict(page_size=8), BAD), (dict(k_pages=0), BAD)])
def test_bad_block_caches_are_refused(change, code):
    for call, name in ((_append, "nmi_kv_append_paged"), (_sparse, "nmi_sdpa_decode_paged_sparse"), (_bounds, "nmi_kv_bounds_paged")):
        assert call(_cache(**change)) == code
        assert _lib.lib().nmi_last_error().decode().startswith(name)


@pytest.mark.parametrize("change,code", [
    (dict(q=0), BAD), (dict(o=0), BAD), (dict(lens=0), BAD), (dict(bounds=0), BAD), (dict(select=0), BAD), (dict(select=-1), BAD),
    (dict(batch=0), BAD), (dict(H=41), BAD), (dict(scale=0.0), BAD), (dict(scale=math.nan), BAD), (dict(batch=2 ** 22), BAD),
    (dict(q=FAKE + 2), ALIGN), (dict(bounds=FAKE + 8), ALIGN), (dict(selected=FAKE + 2), ALIGN), (dict(ws=FAKE + 4), ALIGN),
    (dict(ws_bytes=64), _lib.NMI_ERR_WORKSPACE)])
def test_sparse_decode_refuses(change, code):
    assert _sparse(_cache(), **change) == code and _sparse(None) == BAD
    size = _lib.lib().nmi_sdpa_decode_paged_sparse_workspace_bytes
    assert size(0, 40, 8, 4, 2) == size(1, 41, 8, 4, 2) == size(1, 40, 8, 0, 2) == size(1, 40, 8, 4, 0) == 0


def test_sparse_decode_refuses_more_groups_than_a_launch_has():
    """The choice has 1024 threads for each sequence's KV head, and a launch less than 2^32."""
    assert _sparse(_cache(), batch=2 ** 19, ws_bytes=1 << 40) == BAD
    assert "too many for one launch" in _lib.lib().nmi_last_error().decode()


@pytest.mark.parametrize("change,code", [
    (dict(bounds=0), BAD), (dict(start=0), BAD), (dict(batch=0), BAD), (dict(tokens=0), BAD), (dict(cu=0), BAD),
    (dict(tokens=2 ** 24), BAD), (dict(batch=2 ** 24, tokens=2 ** 24 - 1), BAD), (dict(bounds=FAKE + 8), ALIGN),
    (dict(cu=FAKE + 2), ALIGN), (dict(start=FAKE + 1), ALIGN)])
def test_bounds_refuse(change, code):
    assert _bounds(_cache(), **change) == code and _bounds(None) == BAD


@pytest.mark.parametrize("change,code", [
    *[(dict([(n, 0)]), BAD) for n in ("lens", "table", "free", "count", "start", "kv", "slots", "lens_out", "count_out")],
    (dict(page=8), BAD), (dict(page=24), BAD), (dict(page=1 << 21), BAD), (dict(stride=3), BAD), (dict(max_pages=0), BAD),
    (dict(n_pages=0), BAD), (dict(max_pages=2 ** 26 + 1, stride=2 ** 27), BAD), (dict(batch=0), BAD), (dict(tokens=-1), BAD),
    (dict(tokens=0, cu=0), BAD), (dict(cu=0), BAD), (dict(batch=2 ** 24), BAD), (dict(tokens=2 ** 24), BAD), (dict(slots=FAKE + 4), ALIGN),
    *[(dict([(n, FAKE + 2)]), ALIGN) for n in ("lens", "new", "table", "free", "count", "start", "kv", "cu", "lens_out", "count_out")]])
def test_assign_refuses(change, code):
    assert _assign(**change) == code and _lib.lib().nmi_last_error().decode().startswith("nmi_kv_assign_paged")


def test_append_refuses_more_blocks_than_a_launch_has():
    assert _append(_cache(), tokens=2 ** 24 - 1, batch=2 ** 24) == BAD
    assert "blocks" in _lib.lib().nmi_last_error().decode()


def _tensors(B=3, n_kv=2, H=4, page=32):
    ints = lambda *s: torch.zeros(*s, dtype=torch.int32)  # noqa: E731
    pages = torch.zeros(5, n_kv, page, 128).to(torch.float8_e4m3fn)
    return dict(q=torch.zeros(B, H * 128, dtype=torch.bfloat16), k=torch.zeros(B, n_kv * 128, dtype=torch.bfloat16), k_pages=pages,
                v_pages=pages.clone(), page_table=ints(B, 4), kv_lens=ints(B), start_pos=ints(B), k_scale=torch.ones(5, n_kv, page // 16),
                v_scale=torch.ones(5, n_kv, page // 16), k_bounds=torch.zeros(5, n_kv, 2, 128, dtype=torch.bfloat16))


def _calls(t, **kw):
    scales = dict(k_scale=t["k_scale"], v_scale=t["v_scale"])
    return {"append": lambda: ops.kv_append_paged(t["k"], t["k"], t["k_pages"], t["v_pages"], t["page_table"], t["start_pos"], **scales),
            "decode": lambda: ops.sdpa_decode_paged(t["q"], t["k_pages"], t["v_pages"], t["page_table"], t["kv_lens"], **scales),
            "sparse": lambda: ops.sdpa_decode_paged_sparse(t["q"], t["k_pages"], t["v_pages"], t["page_table"], t["kv_lens"],
                                                           t["k_bounds"], kw.get("n_select", 2), selected=kw.get("selected"), **scales),
            "bounds": lambda: ops.kv_bounds_paged(t["k_pages"], t["page_table"], t["start_pos"], t["k_bounds"],
                                                  k_scale=t["k_scale"], **kw.get("packed", {}))}


def test_front_end_takes_block_scales():
    """Valid calls, refused for nothing but the device."""
    for name, call in _calls(_tensors()).items():
        with pytest.raises(ValueError, match="GPU"):
            call()


@pytest.mark.parametrize("name,value", [
    ("k_scale", torch.ones(5, 2, 1)), ("k_scale", torch.ones(4, 2, 2)), ("k_scale", torch.ones(5, 2, 4)[:, :, ::2]),
    ("k_scale", torch.ones(5, 2, 2).double()), ("k_scale", torch.ones(2))])
def test_front_end_refuses_bad_block_scales(name, value):
    t = _tensors()
    t[name] = value
    for which, call in _calls(t).items():
        if which == "bounds" and value.dim() == 1:
            continue                                     # (a scale per head, as it may be)
        with pytest.raises(ValueError, match="k_scale|v_scale"):
            call()
    t = _tensors()
    t["v_scale"] = None
    with pytest.raises(TypeError, match="v_scale"):
        _calls(t)["decode"]()
    t = _tensors()
    t["k_pages"] = t["v_pages"] = torch.zeros(5, 2, 32, 128, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="bf16 cache"):
        _calls(t)["decode"]()


def test_front_end_refuses_bad_bounds_and_selections():
    for value in (torch.zeros(5, 2, 2, 128), torch.zeros(5, 2, 1, 128, dtype=torch.bfloat16), torch.zeros(5, 2, 256, dtype=torch.bfloat16),
                  torch.zeros(4, 2, 2, 128, dtype=torch.bfloat16), torch.zeros(5, 2, 2, 256, dtype=torch.bfloat16)[..., ::2]):
        t = _tensors()
        t["k_bounds"] = value
        for which in ("sparse", "bounds"):
            with pytest.raises(ValueError, match="k_bounds"):
                _calls(t)[which]()
    t = _tensors()
    for n in (0, -1, 2 ** 31):
        with pytest.raises(ValueError, match="n_select"):
            _calls(t, n_select=n)["sparse"]()
    with pytest.raises(TypeError, match="n_select"):
        _calls(t, n_select=2.5)["sparse"]()
    for selected in (torch.zeros(3, 2, 3, dtype=torch.int32), torch.zeros(3, 2, 2), torch.zeros(3, 2, 4, dtype=torch.int32)[..., ::2]):
        with pytest.raises(ValueError, match="selected"):
            _calls(t, selected=selected)["sparse"]()
    for packed in (dict(tokens=3), dict(cu_seqlens=torch.zeros(4, dtype=torch.int32)),
                   dict(cu_seqlens=torch.zeros(3, dtype=torch.int32), tokens=3), dict(cu_seqlens=torch.zeros(4, dtype=torch.int32), tokens=-1)):
        with pytest.raises(ValueError) as e:
            _calls(t, packed=packed)["bounds"]()
        assert "on a GPU" not in str(e.value)


def test_front_end_refuses_bad_assignments():
    ints = lambda *s: torch.zeros(*s, dtype=torch.int32)  # noqa: E731
    good = dict(lens=ints(3), new_lens=ints(3), page_table=ints(3, 4), free_pages=ints(9), free_count=ints(1), page_size=16)
    with pytest.raises(ValueError, match="GPU"):
        ops.kv_assign_paged(**good)
    with pytest.raises(ValueError, match="GPU"):
        ops.kv_assign_paged(**good, tokens=7, lens_out=good["lens"], free_count_out=good["free_count"])
    for change in (dict(lens=ints(3).long()), dict(lens=ints(3, 1)), dict(new_lens=ints(2)), dict(page_table=ints(2, 4)),
                   dict(page_table=ints(4, 3).t()), dict(page_table=ints(3, 4).long()), dict(free_pages=ints(9, 1)),
                   dict(free_pages=torch.zeros(9)), dict(free_count=ints(2)), dict(page_size=-1), dict(tokens=-1),
                   dict(tokens=2, new_lens=None), dict(lens_out=ints(2)), dict(free_count_out=ints(1).long()),
                   dict(lens_out=good["new_lens"]), dict(lens=ints(0), new_lens=ints(0), page_table=ints(0, 4))):
        with pytest.raises(ValueError) as e:
            ops.kv_assign_paged(**{**good, **change})
        assert "on a GPU" not in str(e.value), change
    for change in (dict(free_count=None), dict(page_size="16"), dict(tokens=1.5), dict(page_table=3)):
        with pytest.raises(TypeError):
            ops.kv_assign_paged(**{**good, **change})


def test_front_end_errors_keep_no_references():
    import sys

    t = _tensors()
    odd = [None, 3, "x", object(), torch.zeros(2, 2).to_sparse(), torch.zeros(()), torch.zeros(0)]
    ints = torch.zeros(3, dtype=torch.int32)
    calls = []
    for which, names in (("append", ("k", "k_pages", "v_pages", "page_table", "start_pos", "k_scale", "v_scale")),
                         ("decode", ("q", "k_pages", "v_pages", "page_table", "kv_lens", "k_scale", "v_scale")),
                         ("sparse", ("q", "k_pages", "page_table", "kv_lens", "k_bounds", "v_scale")),
                         ("bounds", ("k_pages", "page_table", "start_pos", "k_bounds"))):
        for n in names:
            calls.append(lambda x, which=which, n=n: _calls({**t, n: x})[which]())
    calls += [lambda x: ops.kv_assign_paged(x, ints, t["page_table"], ints, ints[:1], 16),
              lambda x: ops.kv_assign_paged(ints, ints, x, ints, ints[:1], 16),
              lambda x: ops.kv_assign_paged(ints, ints, t["page_table"], x, ints[:1], 16),
              lambda x: ops.kv_assign_paged(ints, ints, t["page_table"], ints, x, 16)]
    held = [*odd[3:], *t.values(), ints]
    before = [sys.getrefcount(x) for x in held]
    for _ in range(3):
        for call in calls:
            for x in odd:
                with pytest.raises((ValueError, TypeError, RuntimeError, AttributeError)):
                    call(x)
    del call, x
    assert [sys.getrefcount(x) for x in held] == before
    from nemotron_infer_amd.csrc import front
    for f in (front.kv_assign_paged, front.kv_bounds_paged, front.sdpa_decode_paged_sparse):
        with pytest.raises(TypeError, match="expected"):
            f(1, 2)


def test_oracle_e4m3_values_have_codes():
    lut = e4m3.decode_lut()
    x = paged.round_e4m3(np.random.default_rng(9).standard_normal(2000) * 100)
    assert np.isin(x, lut[np.isfinite(lut)]).all()
