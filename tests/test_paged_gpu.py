"""GPU parity of batched attention serving: appending to a paged KV cache, decode attention over it, and
attention over packed prompts, through the torch front end.

Bars (derived before the first run):
* attention: the parity gate of oracle.linear.parity (2 bf16 ulp, at most 1% one-ulp flips, rel_l2 <=
  1e-3) against float64 rounded once.  The kernels' values differ from the float64 ones by float32
  rounding (2^-24 per operation, sums of at most some thousand terms) and the softmax weights' 16 bits
  (2^-17 each), far below half a bf16 step (2^-9): a value moves to the neighbouring bf16 only from
  next to a border.
* rotation: |kernel - exact| <= d = (|x| + |y|) 2^-20 before rounding (x, y the pair): a float32 angle
  would be off by at most 2^-24 turns half = 1.9e-7 and its sine by 2 ulp = 1.2e-7, 3.1e-7 < 2^-21 on
  each of the two terms (the kernel's are better), their products and sum 3 * 2^-24.  Rounding is monotone, so the output must lie between
  the rounded ends of [exact - d, exact + d].  For e4m3 the same with the division's 2^-24 and the
  scale: d / s + |exact / s| 2^-22.
* what is not rotated and not scaled is copied: bit for bit; what is not addressed stays bit for bit.
"""
import ctypes
import sys
import threading

import numpy as np
import pytest
import torch

from nemotron_infer_amd import _lib, ops
from oracle import block, e4m3, linear, paged
from tests.gpu_util import DEV, announce, assert_parity, bits

pytestmark = pytest.mark.gpu

LUT = e4m3.decode_lut().astype(np.float64)
NAN_BF16 = 0x7FC0


@pytest.fixture(autouse=True)
def _no_pending_error():
    _lib.lib().nmi_async_status()
    yield
    torch.cuda.synchronize()
    _lib.lib().nmi_async_status()


def _rand_bits(rng, *shape, scale=1.0):
    return block.bf16_round_exact(rng.standard_normal(shape) * scale)


def _dev(x):
    x = np.ascontiguousarray(x)
    if x.dtype == np.uint16:
        return torch.from_numpy(x.view(np.int16)).view(torch.bfloat16).to(DEV)
    if x.dtype == np.int64:
        x = x.astype(np.int32)
    return torch.from_numpy(x).to(DEV)


def _f64(b):
    return linear.bf16_to_f32(np.asarray(b, np.uint16)).astype(np.float64)


class Pool:
    """A pool of pages with the sequences' pages scattered over it; on the host and on the GPU.  What lies
    behind a sequence's length, and in pages of nobody, is NaN."""

    def __init__(self, rng, lens, n_kv, page, kind, layout="heads", extra=3, width=None, hold=None):
        hold = lens if hold is None else hold              # positions that the pages must be able to hold
        counts = [-(-int(max(0, n)) // page) for n in hold]
        n_pages = sum(counts) + extra
        width = max(1, max(counts)) + 1 if width is None else width
        ids = rng.permutation(n_pages)
        self.table = np.full((len(lens), width), -1, np.int32)
        at = 0
        for b, c in enumerate(counts):
            self.table[b, :c] = ids[at:at + c]
            at += c
        self.page, self.n_kv, self.kind, self.lens = page, n_kv, kind, np.array(lens, np.int32)
        shape = (n_pages, n_kv, page, 128)
        if kind == "bf16":
            self.k, self.v = np.full(shape, NAN_BF16, np.uint16), np.full(shape, NAN_BF16, np.uint16)
            make = lambda *s: _rand_bits(rng, *s)  # noqa: E731
            self.ks = self.vs = None
        else:
            self.k, self.v = np.full(shape, 0x7F, np.uint8), np.full(shape, 0x7F, np.uint8)
            make = lambda *s: e4m3.quantize_rne(np.clip(rng.standard_normal(s) * 60, -448, 448))  # noqa: E731
            self.ks, self.vs = (rng.uniform(0.01, 0.03, n_kv).astype(np.float32) for _ in range(2))
        for b, n in enumerate(self.lens):
            for p0 in range(0, max(0, n), page):
                m = min(page, n - p0)
                for pool in (self.k, self.v):
                    pool[self.table[b, p0 // page], :, :m] = make(n_kv, m, 128)
        self.layout = layout
        self.dk, self.dv = self._to_dev(self.k), self._to_dev(self.v)
        self.dtable = _dev(self.table)
        self.dks, self.dvs = (None if s is None else _dev(s) for s in (self.ks, self.vs))

    def _to_dev(self, x):
        if self.layout == "tokens":                        # [n_pages, page, n_kv, 128] seen as the other
            return _dev(x.transpose(0, 2, 1, 3)).transpose(1, 2)
        if self.layout == "slice":                         # one layer of a pool of three, K and V side by side
            big = torch.zeros((x.shape[0], 3) + x.shape[1:], dtype=_dev(x[:1]).dtype, device=DEV)
            big[:, 1] = _dev(x)
            return big[:, 1]
        return _dev(x)

    def values(self):
        if self.kind == "bf16":
            return _f64(self.k), _f64(self.v)
        return (LUT[self.k] * self.ks.astype(np.float64)[:, None, None],
                LUT[self.v] * self.vs.astype(np.float64)[:, None, None])

    def decode(self, q, lens=None, **kw):
        lens = _dev(self.lens if lens is None else np.array(lens, np.int32))
        return ops.sdpa_decode_paged(q, self.dk, self.dv, self.dtable, lens, k_scale=self.dks, v_scale=self.dvs, **kw)

    def host(self, t):
        """A pool on the GPU as bits [n_pages, n_kv, page, 128]."""
        t = t.contiguous()
        return bits(t) if self.kind == "bf16" else t.cpu().numpy()


def _check_decode(rng, lens, H, n_kv, page, kind, qscale=1.0, label="", scale=None, **kw):
    pool = Pool(rng, lens, n_kv, page, kind, **kw)
    q = _rand_bits(rng, len(lens), H * 128, scale=qscale)
    o = pool.decode(_dev(q), **({} if scale is None else {"scale": scale}))
    torch.cuda.synchronize()
    K, V = pool.values()
    want = paged.decode(_f64(q).reshape(len(lens), H, 128), K, V, pool.table, pool.lens,
                        **({} if scale is None else {"scale": scale}))
    got = bits(o).reshape(want.shape)
    for b, n in enumerate(pool.lens):
        if n <= 0:
            assert not got[b].any(), f"{label}: length {n}"
    live = pool.lens > 0
    if live.any():
        assert_parity(got[live], block.bf16_round_exact(want[live]), label)
    assert _lib.lib().nmi_async_status() == 0
    return o


# --- decode ----------------------------------------------------------------------------------------


@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
@pytest.mark.parametrize("n", [0, 1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 200, 777, 1025])
def test_decode_lengths(kind, n):
    announce("paged_decode", kind, n)
    _check_decode(np.random.default_rng(n), [n], 40, 8, 16, kind, label=f"{kind} {n}")


@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
@pytest.mark.parametrize("H,n_kv", [(1, 1), (8, 8), (6, 2), (7, 1), (16, 1), (17, 1), (40, 1), (66, 2), (32, 4)])
def test_decode_head_groups(kind, H, n_kv):
    announce("paged_heads", kind, H, n_kv)
    _check_decode(np.random.default_rng(H * 100 + n_kv), [45, 0, 300, 1], H, n_kv, 32, kind, label=f"{H}/{n_kv}")


@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
@pytest.mark.parametrize("page", [16, 32, 64, 256, 1024])
@pytest.mark.parametrize("layout", ["heads", "tokens", "slice"])
def test_decode_pages_and_layouts(kind, page, layout):
    announce("paged_layout", kind, page, layout)
    _check_decode(np.random.default_rng(page), [70, 513, 16, 1300], 16, 4, page, kind, label=f"{page} {layout}",
                  layout=layout)


@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
def test_decode_ragged_batches(kind):
    """More sequences than lanes, idle ones and negative lengths among them; one long one among short ones."""
    rng = np.random.default_rng(7)
    for lens in ([int(n) for n in rng.integers(0, 90, 64)], [int(n) for n in rng.integers(-3, 60, 150)],
                 [3] * 70 + [5000] + [17] * 60, [0] * 5):
        announce("paged_ragged", kind, len(lens), max(lens))
        _check_decode(rng, lens, 8, 2, 16, kind, label=f"{len(lens)} sequences")


@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
@pytest.mark.parametrize("batch", [65, 128, 129, 320, 321, 700])
def test_decode_many_sequences(kind, batch):
    announce("decode_many", kind, batch)
    rng = np.random.default_rng(batch)
    lens = rng.integers(1, 60, batch)
    lens[rng.integers(0, batch, batch // 4)] = 0
    lens[[batch // 3, batch - 1]] = 700, 333
    _check_decode(rng, lens, 4, 2, 16, kind, label=f"{batch} sequences")


@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
def test_decode_long_peaked_flat_and_scaled(kind):
    rng = np.random.default_rng(8)
    announce("paged_long", kind)
    _check_decode(rng, [20000, 33], 10, 2, 128, kind, label="long")
    announce("paged_peaked", kind)
    _check_decode(rng, [700, 90], 10, 2, 16, kind, qscale=8.0, label="peaked")
    _check_decode(rng, [700, 90], 10, 2, 16, kind, qscale=0.0, label="flat")
    _check_decode(rng, [700, 90], 10, 2, 16, kind, scale=0.5, label="scale 0.5")
    _check_decode(rng, [700, 90], 10, 2, 16, kind, scale=1e-3, label="scale 1e-3")


def test_decode_offsets_past_32_bits():
    """Two pages 6 GiB apart in one pool (the stride between pages is the pool's own)."""
    announce("paged_far")
    rng = np.random.default_rng(9)
    far = 3 << 30                                          # elements
    store = torch.empty(far + 2 * 16 * 128, dtype=torch.bfloat16, device=DEV)
    pages = torch.as_strided(store, (2, 2, 16, 128), (far, 16 * 128, 128, 1))
    kb, vb = _rand_bits(rng, 2, 2, 16, 128), _rand_bits(rng, 2, 2, 16, 128)
    pages.copy_(_dev(kb))
    store_v = torch.empty_like(store)
    v_pages = torch.as_strided(store_v, (2, 2, 16, 128), (far, 16 * 128, 128, 1))
    v_pages.copy_(_dev(vb))
    q = _rand_bits(rng, 1, 4 * 128)
    table = np.array([[1, 0]], np.int32)
    o = ops.sdpa_decode_paged(_dev(q), pages, v_pages, _dev(table), _dev(np.array([27], np.int32)))
    want = paged.decode(_f64(q).reshape(1, 4, 128), _f64(kb), _f64(vb), table, [27])
    assert_parity(bits(o).reshape(want.shape), block.bf16_round_exact(want), "far pages")
    kn, vn = _rand_bits(rng, 1, 2 * 128), _rand_bits(rng, 1, 2 * 128)
    ops.kv_append_paged(_dev(kn), _dev(vn), pages, v_pages, _dev(table[:, ::-1].copy()), _dev(np.array([20], np.int32)))
    kb[1, :, 4], vb[1, :, 4] = kn.reshape(2, 128), vn.reshape(2, 128)
    assert np.array_equal(bits(pages.contiguous()), kb) and np.array_equal(bits(v_pages.contiguous()), vb)


def test_decode_of_sequences_that_share_pages():
    """A page in several sequences' tables, and twice in one: the same positions read by all of them."""
    announce("decode_shared_pages")
    rng = np.random.default_rng(12)
    pool = Pool(rng, [640, 64], 2, 16, "bf16")
    pool.table = np.stack([pool.table[0], pool.table[0], np.where(np.arange(pool.table.shape[1]) % 2, pool.table[1, 1], pool.table[0, 3])])
    pool.dtable, pool.lens = _dev(pool.table), np.array([640, 333, 600], np.int32)
    q = _rand_bits(rng, 3, 8 * 128)
    o = pool.decode(_dev(q))
    torch.cuda.synchronize()
    K, V = pool.values()
    want = paged.decode(_f64(q).reshape(3, 8, 128), K, V, pool.table, pool.lens)
    assert_parity(bits(o).reshape(want.shape), block.bf16_round_exact(want), "shared pages")


def test_decode_takes_its_workspace_from_the_allocator():
    """Through the C ABI without a workspace."""
    announce("decode_bump")
    rng = np.random.default_rng(13)
    pool = Pool(rng, [900, 5], 4, 16, "e4m3")
    q = _dev(_rand_bits(rng, 2, 16 * 128))
    want, got = pool.decode(q), torch.zeros(2, 16 * 128, dtype=torch.bfloat16, device=DEV)
    L, lens = _lib.lib(), _dev(pool.lens)
    c = _lib.PagedKv(pool.dk.data_ptr(), pool.dv.data_ptr(), 4 * 16 * 128, 16 * 128, 128, pool.dtable.data_ptr(),
                     pool.table.shape[1], pool.dks.data_ptr(), pool.dvs.data_ptr(), 1, pool.dk.shape[0], 16,
                     pool.table.shape[1], 4)
    for _ in range(2):
        got.zero_()
        rc = L.nmi_sdpa_decode_paged(ctypes.addressof(c), q.data_ptr(), 16 * 128, got.data_ptr(), 16 * 128, lens.data_ptr(), 2,
                                     16, 128 ** -0.5, None, 0, torch.cuda.current_stream().cuda_stream)
        assert rc == 0, L.nmi_last_error()
        torch.cuda.synchronize()
        assert torch.equal(got.view(torch.int16), want.view(torch.int16))
        assert L.nmi_alloc_rewind() in (0, None)


def test_decode_strides_and_outputs():
    """q and o as columns of wider buffers; the rest of o's buffer stays as it was."""
    announce("paged_strides")
    rng = np.random.default_rng(10)
    pool = Pool(rng, [100, 5, 40], 2, 16, "bf16")
    q = _rand_bits(rng, 3, 8 * 128)
    wide = torch.full((3, 8 * 128 + 72), 9.0, dtype=torch.bfloat16, device=DEV)
    wide[:, 8:8 + 1024] = _dev(q)
    out = torch.full((3, 8 * 128 + 6), 7.0, dtype=torch.bfloat16, device=DEV)
    pool.decode(wide[:, 8:8 + 1024], out=out[:, 2:1026])
    alone = pool.decode(_dev(q))
    assert torch.equal(out[:, 2:1026].view(torch.int16), alone.view(torch.int16))
    assert (out[:, :2] == 7).all() and (out[:, 1026:] == 7).all()


@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
def test_decode_is_the_same_every_time(kind):
    announce("paged_repeat", kind)
    rng = np.random.default_rng(11)
    pool = Pool(rng, [3000, 17, 900], 8, 64, kind)
    q = _dev(_rand_bits(rng, 3, 40 * 128))
    first = pool.decode(q)
    for _ in range(5):
        assert torch.equal(pool.decode(q).view(torch.int16), first.view(torch.int16))


def test_decode_equals_the_contiguous_operator():
    """Against nmi_sdpa_decode_bf16 over the same positions: the same gate as against the oracle, since
    each is float32 in an order of its own."""
    announce("paged_vs_contiguous")
    rng = np.random.default_rng(12)
    pool = Pool(rng, [513], 8, 16, "bf16")
    q = _rand_bits(rng, 1, 40 * 128)
    kc, vc = (torch.cat([p[i] for i in pool.table[0, :33]], dim=1) for p in (pool.dk, pool.dv))
    kc, vc = torch.nan_to_num(kc).contiguous(), torch.nan_to_num(vc).contiguous()
    new = torch.zeros(8, 128, dtype=torch.bfloat16, device=DEV)
    old = ops.sdpa_decode_bf16(_dev(q).view(40, 128), kc, vc, new, new, 513)
    assert_parity(bits(pool.decode(_dev(q))).reshape(40, 128), bits(old), "contiguous")


def test_decode_bad_pages_and_lengths_are_reported():
    """A page outside the pool or a length past the table: NaN in that sequence, the others right, and
    one NMI_ERR_ASYNC; the next call works."""
    rng = np.random.default_rng(13)
    for change in ("page", "negative", "length"):
        announce("paged_bad", change)
        pool = Pool(rng, [90, 200, 40], 2, 16, "bf16")
        q = _rand_bits(rng, 3, 8 * 128)
        good = bits(pool.decode(_dev(q)))
        lens = pool.lens.copy()
        if change == "length":
            lens[1] = pool.table.shape[1] * 16 + 1
        else:
            table = pool.table.copy()
            table[1, 3] = pool.k.shape[0] if change == "page" else -1
            pool.dtable = _dev(table)
        got = bits(pool.decode(_dev(q), lens=lens))
        torch.cuda.synchronize()
        assert np.isnan(_f64(got[1])).all()
        assert np.array_equal(got[[0, 2]], good[[0, 2]])
        pool.dtable = _dev(pool.table)
        with pytest.raises(_lib.NmiError) as e:
            pool.decode(_dev(q))
        assert e.value.code == _lib.NMI_ERR_ASYNC and "page" in str(e.value)
        assert np.array_equal(bits(pool.decode(_dev(q))), good)


# --- append ----------------------------------------------------------------------------------------


def _between(got, exact, d, rounded):
    """got lies between the rounded ends of [exact - d, exact + d]."""
    lo, hi = rounded(exact - d), rounded(exact + d)
    bad = ~((lo <= got) & (got <= hi))
    assert not bad.any(), (int(bad.sum()), got[bad][:4], exact[bad][:4])


def _bf16(x):
    return _f64(block.bf16_round_exact(x))


def _check_append(rng, starts, lens, H, n_kv, page, kind, rotary, interleaved, with_q=True, with_k=True, in_place=False,
                  layout="heads", lead=0, tail=0, packed=True, theta=10000.0):
    starts = np.array(starts, np.int32)
    T = lead + sum(lens) + tail
    cu = lead + np.concatenate([[0], np.cumsum(lens)]).astype(np.int32)
    hold = [max(0, int(s)) + n for s, n in zip(starts, lens)]
    pool = Pool(rng, [max(0, int(s)) for s in starts], n_kv, page, kind, layout=layout, hold=hold)
    buf = _rand_bits(rng, T, (H + 2 * n_kv) * 128)
    dbuf = _dev(buf)
    cols = [0, H * 128, (H + n_kv) * 128, (H + 2 * n_kv) * 128]
    dq, dk, dv = (dbuf[:, a:b] for a, b in zip(cols, cols[1:]))
    q, k, v = (_f64(buf[:, a:b]).reshape(T, -1, 128) for a, b in zip(cols, cols[1:]))
    f = None
    if rotary:
        f = (theta ** (-np.arange(rotary // 2) / (rotary // 2))).astype(np.float32)
    with_q, with_k = with_q and rotary > 0, with_k and rotary > 0
    qo = (dq if in_place else torch.full((T, H * 128), 5.0, dtype=torch.bfloat16, device=DEV)) if with_q else None
    ko = (dk if in_place else torch.full((T, n_kv * 128), 5.0, dtype=torch.bfloat16, device=DEV)) if with_k else None
    before = [pool.host(pool.dk).copy(), pool.host(pool.dv).copy()]
    got_q, got_k = ops.kv_append_paged(dk, dv, pool.dk, pool.dv, pool.dtable, _dev(starts),
                                       cu_seqlens=_dev(cu) if packed else None, q=dq if with_q else None,
                                       inv_freq=None if f is None else _dev(f), interleaved=interleaved,
                                       k_scale=pool.dks, v_scale=pool.dvs, q_out=qo, k_out=ko)
    torch.cuda.synchronize()
    assert _lib.lib().nmi_async_status() == 0
    assert got_q is qo and got_k is ko
    rows = paged.positions(T, starts, cu if packed else None)
    if not rows:
        assert np.array_equal(pool.host(pool.dk), before[0]) and np.array_equal(pool.host(pool.dv), before[1])
        return
    r, seq, pos = (np.array(x) for x in zip(*rows))
    at = (pool.table[seq, pos // page], slice(None), pos % page)
    if rotary:
        eq, ek = (paged.rotate(x[r], pos.astype(np.float64), f, interleaved) for x in (q, k))
        pq, pk = (paged.partner_sum(x[r], rotary, interleaved) * 2.0 ** -20 for x in (q, k))
    else:
        ek, pk = k[r], np.zeros_like(k[r])
    untouched = np.setdiff1d(np.arange(T), r)
    for out, src, exact, d, given in ((qo, buf[:, :cols[1]], eq if rotary else None, pq if rotary else None, with_q),
                                      (ko, buf[:, cols[1]:cols[2]], ek, pk, with_k)):
        if given:
            host = bits(out)
            _between(_f64(host[r]).reshape(exact.shape), exact, d, _bf16)
            left = src[untouched] if in_place else np.full_like(src[untouched], bits(torch.full((1,), 5.0).bfloat16())[0])
            assert np.array_equal(host[untouched], left)
    for name, dpool, old, exact, d, s in (("k", pool.dk, before[0], ek, pk, pool.ks),
                                          ("v", pool.dv, before[1], v[r], 0 * v[r], pool.vs)):
        new = pool.host(dpool)
        if kind == "bf16":
            if not rotary or name == "v":
                assert np.array_equal(_f64(new[at]), exact)
            else:
                _between(_f64(new[at]), exact, d, _bf16)
        else:
            sc = s.astype(np.float64)[:, None]
            _between(LUT[new[at]], exact / sc, d / sc + np.abs(exact / sc) * 2.0 ** -22, paged.round_e4m3)
        mask = np.ones(new.shape, bool)
        mask[at] = False
        assert np.array_equal(new[mask], old[mask]), f"{name}: other places changed"


@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
@pytest.mark.parametrize("rotary,interleaved", [(0, False), (128, False), (128, True), (64, False), (16, True), (112, False), (96, True)])
def test_append_prompts(kind, rotary, interleaved):
    announce("append", kind, rotary, interleaved)
    rng = np.random.default_rng(rotary)
    _check_append(rng, [0, 5, 31, 0, 100], [70, 1, 33, 0, 16], 8, 2, 32, kind, rotary, interleaved)
    _check_append(rng, [7, 0], [20, 3], 5, 5, 16, kind, rotary, interleaved, layout="tokens", lead=2, tail=3)


@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
@pytest.mark.parametrize("batch", [1, 3, 64, 65, 200])
def test_append_one_token_each(kind, batch):
    announce("append_decode", kind, batch)
    rng = np.random.default_rng(batch)
    starts = rng.integers(0, 300, batch)
    starts[batch // 2] = -1 if batch > 1 else 40                    # a sequence that is not in use
    for packed in (False, True):
        _check_append(rng, starts, [1] * batch, 6, 2, 16, kind, 128, False, packed=packed, in_place=not packed)


def test_append_many_sequences_of_odd_lengths():
    announce("append_many")
    rng = np.random.default_rng(20)
    lens = [int(n) for n in rng.integers(0, 5, 300)]
    _check_append(rng, [int(s) for s in rng.integers(-2, 40, 300)], lens, 4, 1, 16, "bf16", 32, True, lead=1, tail=70)


@pytest.mark.parametrize("kind,rotary,interleaved", [("bf16", 0, False), ("bf16", 128, False), ("e4m3", 96, True)])
def test_append_more_vectors_than_a_wave_loads_at_once(kind, rotary, interleaved):
    """A wave for a token, whose head vectors it takes in two turns; in place, too."""
    announce("append_turns", kind, rotary)
    rng = np.random.default_rng(23)
    _check_append(rng, [3, 0, 90], [600, 37, 700], 48, 16, 32, kind, rotary, interleaved, in_place=rotary > 0, lead=1, tail=1)


def test_append_offsets_past_32_bits():
    """Pages whose bytes lie more than 2^32 from the pool's start."""
    announce("append_large_pool")
    n_pages, n_kv, page = 70000, 8, 32
    k_pages = torch.empty(n_pages, n_kv, page, 128, dtype=torch.bfloat16, device=DEV)
    v_pages = torch.empty_like(k_pages)
    assert k_pages.numel() * 2 > 1 << 32
    rng = np.random.default_rng(24)
    k, v = (_rand_bits(rng, 40, n_kv * 128) for _ in range(2))
    table = np.array([[n_pages - 1, 66001], [65999, n_pages - 2]], np.int32)
    for t in table.flat:
        k_pages[int(t)].zero_(), v_pages[int(t)].zero_()
    ops.kv_append_paged(_dev(k), _dev(v), k_pages, v_pages, _dev(table), _dev(np.array([20, 31], np.int32)),
                        cu_seqlens=_dev(np.array([0, 30, 40], np.int32)))
    torch.cuda.synchronize()
    for x, pool in ((k, k_pages), (v, v_pages)):
        want = {int(t): np.zeros((n_kv, page, 128), np.uint16) for t in table.flat}
        for t in range(40):
            b, pos = (0, 20 + t) if t < 30 else (1, 31 + t - 30)
            want[int(table[b, pos // page])][:, pos % page] = x[t].reshape(n_kv, 128)
        for i, w in want.items():
            assert np.array_equal(bits(pool[i]), w), i


def test_append_at_far_positions():
    """Angles of positions in the hundreds of thousands, at full accuracy."""
    announce("append_far")
    rng = np.random.default_rng(21)
    for starts in ([131071, 999983], [10 ** 6 + 7, 3]):
        _check_append_far(rng, starts)


def _check_append_far(rng, starts):
    n_kv, page, rotary = 2, 1024, 128
    table = np.zeros((2, 1024), np.int32)
    table[0, starts[0] // page], table[1, starts[1] // page] = 1, 0
    pages = [torch.zeros(2, n_kv, page, 128, dtype=torch.bfloat16, device=DEV) for _ in range(2)]
    q, k, v = _rand_bits(rng, 2, 4 * 128), _rand_bits(rng, 2, n_kv * 128), _rand_bits(rng, 2, n_kv * 128)
    f = (10000.0 ** (-np.arange(64) / 64)).astype(np.float32)
    q_out, _ = ops.kv_append_paged(_dev(k), _dev(v), *pages, _dev(table), _dev(np.array(starts, np.int32)), q=_dev(q),
                                   inv_freq=_dev(f))
    pos = np.array(starts, np.float64)
    x = _f64(q).reshape(2, 4, 128)
    _between(_f64(bits(q_out)).reshape(x.shape), paged.rotate(x, pos, f, False),
             paged.partner_sum(x, rotary, False) * 2.0 ** -20, _bf16)
    x = _f64(k).reshape(2, n_kv, 128)
    got = np.stack([_f64(bits(pages[0]))[1 - b, :, starts[b] % page] for b in range(2)])
    _between(got, paged.rotate(x, pos, f, False), paged.partner_sum(x, rotary, False) * 2.0 ** -20, _bf16)


def test_append_e4m3_saturates_and_keeps_nan():
    announce("append_saturates")
    vals = np.array([0.0, -0.0, 448.0, 449.0, 463.9, 464.0, 1000.0, -1e30, 3e38, np.inf, -np.inf, np.nan, 2.0 ** -9, 2.0 ** -10,
                     2.0 ** -11, 1.5 * 2.0 ** -9, 17.0, 18.0, 19.0, -21.0])
    x = np.zeros((1, 128))
    x[0, :len(vals)] = vals
    xb = block.bf16_round_exact(x)
    xb[0, 11] = NAN_BF16
    pages = [torch.zeros(1, 1, 16, 128, dtype=torch.float8_e4m3fn, device=DEV) for _ in range(2)]
    ops.kv_append_paged(_dev(xb), _dev(xb), *pages, _dev(np.zeros((1, 1), np.int32)), _dev(np.array([3], np.int32)))
    want = paged.round_e4m3(_f64(xb)[0])
    for p in pages:
        got = LUT[p.view(torch.uint8).cpu().numpy()[0, 0, 3]]
        assert np.array_equal(got, want, equal_nan=True), (got[:20], want[:20])


def test_append_bad_places_are_skipped_and_reported():
    """A position past the table or a page outside the pool: that token is not stored, its rotated q is
    still right, the others are stored, and NMI_ERR_ASYNC says so once."""
    rng = np.random.default_rng(22)
    f = _dev(np.ones(8, np.float32))
    for table, starts in (([[0], [-1], [1]], [3, 4, 5]), ([[0], [2], [1]], [3, 4, 5]), ([[0], [0], [1]], [3, 16, 5]),
                          ([[0], [0], [1]], [3, 2 ** 31 - 1, 5])):
        announce("append_bad", table, starts)
        pages = [torch.zeros(2, 1, 16, 128, dtype=torch.bfloat16, device=DEV) for _ in range(2)]
        k, v, q = (_dev(_rand_bits(rng, 3, 128)) for _ in range(3))
        q_out, _ = ops.kv_append_paged(k, v, *pages, _dev(np.array(table, np.int32)), _dev(np.array(starts, np.int32)), q=q,
                                       inv_freq=f)
        torch.cuda.synchronize()
        assert torch.equal(pages[1][0, 0, 3], v[0]) and torch.equal(pages[1][1, 0, 5], v[2])
        assert int((pages[1].abs().sum(-1) > 0).sum()) == 2
        assert q_out.abs().sum(-1).min() > 0
        assert _lib.lib().nmi_async_status() == _lib.NMI_ERR_ASYNC
        assert _lib.lib().nmi_async_status() == 0


# --- packed prompts --------------------------------------------------------------------------------


def _check_prefill(rng, lens, H, n_kv, lead=0, tail=0, qscale=1.0, scale=None, poison=True, wide=False):
    T = lead + sum(lens) + tail
    cu = lead + np.concatenate([[0], np.cumsum(lens)]).astype(np.int32)
    q, k, v = _rand_bits(rng, T, H * 128, scale=qscale), _rand_bits(rng, T, n_kv * 128), _rand_bits(rng, T, n_kv * 128)
    outside = np.r_[0:lead, T - tail:T]
    if poison:
        for x in (q, k, v):
            x[outside] = NAN_BF16
    dq, dk, dv = _dev(q), _dev(k), _dev(v)
    if wide:
        buf = torch.cat([dq, dk, dv], dim=1)
        dq, dk, dv = buf[:, :H * 128], buf[:, H * 128:(H + n_kv) * 128], buf[:, (H + n_kv) * 128:]
    out = torch.full((T, H * 128 + (12 if wide else 0)), 3.0, dtype=torch.bfloat16, device=DEV)
    kw = {} if scale is None else {"scale": scale}
    ops.sdpa_prefill_packed_bf16(dq, dk, dv, _dev(cu), H, n_kv, out=out, **kw)
    torch.cuda.synchronize()
    assert _lib.lib().nmi_async_status() == 0
    got = out[:, :H * 128]
    assert (out[outside] == 3).all() and (out[:, H * 128:] == 3).all()
    want = paged.prefill(_f64(q).reshape(T, H, 128), _f64(k).reshape(T, n_kv, 128), _f64(v).reshape(T, n_kv, 128), cu, **kw)
    inside = slice(lead, T - tail)
    assert_parity(bits(got.contiguous()).reshape(want.shape)[inside], block.bf16_round_exact(want[inside]), f"{lens[:8]}")
    return got


@pytest.mark.parametrize("n", [1, 2, 31, 32, 33, 63, 64, 65, 127, 128, 129, 200, 257, 400])
def test_prefill_one_length(n):
    announce("packed", n)
    rng = np.random.default_rng(n)
    _check_prefill(rng, [n], 4, 2)
    _check_prefill(rng, [n, 1, n], 2, 1, lead=3, tail=5)


@pytest.mark.parametrize("lens", [[0, 5, 0, 130, 0], [700, 3, 260], [1] * 70, [129, 128, 127, 1, 64, 300, 65],
                                  [0] * 65 + [200] + [0] * 70 + [131, 7], [16] * 130])
def test_prefill_ragged(lens):
    announce("packed_ragged", len(lens), sum(lens))
    _check_prefill(np.random.default_rng(sum(lens)), lens, 6, 2, lead=1, tail=2, wide=True)


@pytest.mark.parametrize("H,n_kv", [(10, 2), (16, 2)])
@pytest.mark.parametrize("lens", [[1, 33, 65, 0, 129, 32, 64, 40, 300, 2] * 33, [65] * 257, [33] * 300, [1] * 600],
                         ids=["ragged", "65", "33", "1"])
def test_prefill_many_sequences(H, n_kv, lens):
    """More sequences than stay at hand, and the lengths that need the most workgroups for their rows."""
    announce("packed_many", H, n_kv, len(lens), sum(lens))
    _check_prefill(np.random.default_rng(len(lens)), lens, H, n_kv, lead=2, tail=1)


def test_prefill_heads_scales_and_peaks():
    rng = np.random.default_rng(31)
    for H, n_kv in ((1, 1), (5, 5), (40, 8), (17, 1)):
        announce("packed_heads", H, n_kv)
        _check_prefill(rng, [70, 20], H, n_kv)
    _check_prefill(rng, [150, 40], 4, 2, qscale=8.0)
    _check_prefill(rng, [150, 40], 4, 2, qscale=0.0)
    _check_prefill(rng, [150, 40], 4, 2, scale=0.3)


@pytest.mark.parametrize("H,n_kv", [(16, 4), (40, 8), (16, 2), (48, 16), (8, 8), (32, 1), (40, 4), (10, 2), (7, 1)])
def test_prefill_equals_the_single_prompt_operator(H, n_kv):
    """A packed prompt gets the bytes that nmi_sdpa_prefill_bf16 gives it alone, whichever heads its last
    rows share a workgroup with: the same kernel body."""
    announce("packed_vs_single", H, n_kv)
    rng = np.random.default_rng(32)
    lens = [300, 1, 1000, 129, 32, 33, 64, 65, 160, 0, 161, 192, 193, 31]
    T = sum(lens)
    q, k, v = _dev(_rand_bits(rng, T, H * 128)), _dev(_rand_bits(rng, T, n_kv * 128)), _dev(_rand_bits(rng, T, n_kv * 128))
    cu = np.concatenate([[0], np.cumsum(lens)]).astype(np.int32)
    got = ops.sdpa_prefill_packed_bf16(q, k, v, _dev(cu), H, n_kv)
    for a, b in zip(cu, cu[1:]):
        if a == b:
            continue
        one = ops.sdpa_prefill_bf16(q[a:b].contiguous(), k[a:b].contiguous(), v[a:b].contiguous(), H, n_kv)
        assert torch.equal(got[a:b].view(torch.int16), one.view(torch.int16)), (a, b)


@pytest.mark.parametrize("bad", [NAN_BF16, 0x7F80, 0xFF80])
def test_prefill_values_that_are_not_finite_stay_with_the_rows_that_see_them(bad):
    """NaN or an infinity in k and v of some keys: the rows before them, and the other prompts, as without."""
    announce("packed_not_finite", hex(bad))
    rng = np.random.default_rng(34)
    H, n_kv, lens = 10, 2, [200, 40, 33, 300]
    T, cu = sum(lens), np.concatenate([[0], np.cumsum(lens)]).astype(np.int32)
    q, k, v = (_rand_bits(rng, T, n * 128) for n in (H, n_kv, n_kv))
    for at in ([199], [77, 150], [200 + 17], [273 + 128]):
        k2, v2 = k.copy(), v.copy()
        for t in at:
            v2[t, rng.integers(0, 128, 5)] = bad                # some dims of KV head 0
            k2[t, 128:] = bad                                   # all of KV head 1
        o = ops.sdpa_prefill_packed_bf16(_dev(q), _dev(k2), _dev(v2), _dev(cu), H, n_kv)
        torch.cuda.synchronize()
        with np.errstate(all="ignore"):
            want = paged.prefill(_f64(q).reshape(T, H, 128), _f64(k2).reshape(T, n_kv, 128), _f64(v2).reshape(T, n_kv, 128), cu)
        got = _f64(bits(o)).reshape(T, H, 128)
        seen = np.zeros(T, bool)
        for t in at:
            seen[t:cu[np.searchsorted(cu, t, side="right")]] = True
        # (an infinite weight or one that underflows times an infinity may be NaN on one side: not finite on both)
        assert np.array_equal(np.isfinite(got[:, :5]), np.isfinite(want[:, :5]))
        assert np.isfinite(got[~seen]).all()
        clean = np.isfinite(got) & np.isfinite(want)
        assert_parity(bits(o).reshape(T, H, 128)[clean], block.bf16_round_exact(want[clean]), f"not finite at {at}")


def test_prefill_rows_far_apart():
    """The largest row stride: offsets past 32 bits within a sequence."""
    announce("packed_far_rows")
    rng = np.random.default_rng(35)
    lens, H, n_kv, ld = [150, 40], 2, 1, 1 << 24
    T, cu = sum(lens), np.array([0, 150, 190], np.int32)
    buf = torch.empty(T * ld, dtype=torch.bfloat16, device=DEV)
    views, host = [], []
    for at, n in ((0, H), (4096, n_kv), (ld - 128, n_kv), (8192, H)):
        views.append(buf.as_strided((T, n * 128), (ld, 1), at))
        host.append(_rand_bits(rng, T, n * 128))
        views[-1].copy_(_dev(host[-1]))
    ops.sdpa_prefill_packed_bf16(*views[:3], _dev(cu), H, n_kv, out=views[3])
    torch.cuda.synchronize()
    q, k, v = (_f64(x).reshape(T, -1, 128) for x in host[:3])
    want = paged.prefill(q, k, v, cu)
    assert_parity(bits(views[3].contiguous()).reshape(want.shape), block.bf16_round_exact(want), "far rows")


def test_prefill_replays_with_other_offsets():
    """One graph, replayed with offsets that change on the device, gives the eager bytes each time; rows of
    no sequence stay."""
    announce("packed_graph")
    rng = np.random.default_rng(36)
    H, n_kv, T = 16, 4, 700
    q, k, v = (_dev(_rand_bits(rng, T, n * 128)) for n in (H, n_kv, n_kv))
    cu = _dev(np.array([0, 700, 700, 700, 700], np.int32))
    out = torch.zeros(T, H * 128, dtype=torch.bfloat16, device=DEV)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        ops.sdpa_prefill_packed_bf16(q, k, v, cu, H, n_kv, out=out)
    for offsets in ([0, 700, 700, 700, 700], [0, 1, 2, 3, 4], [5, 5, 260, 261, 699], [0, 128, 256, 384, 512], [9, 9, 9, 9, 9]):
        cu.copy_(_dev(np.array(offsets, np.int32)))
        out.fill_(3.0)
        g.replay()
        eager = ops.sdpa_prefill_packed_bf16(q, k, v, cu, H, n_kv, out=torch.full_like(out, 3.0))
        torch.cuda.synchronize()
        assert torch.equal(out.view(torch.int16), eager.view(torch.int16)), offsets
        rest = torch.ones(T, dtype=torch.bool)
        rest[offsets[0]:offsets[-1]] = False
        assert (out.cpu()[rest] == 3.0).all()
    assert _lib.lib().nmi_async_status() == 0


def test_nothing_to_do():
    """No sequences, or no rows: nothing is launched, the outputs are empty."""
    announce("paged_empty")
    pool = Pool(np.random.default_rng(37), [3], 2, 16, "bf16")
    rows = lambda n: torch.empty(0, n * 128, dtype=torch.bfloat16, device=DEV)  # noqa: E731
    none = torch.empty(0, dtype=torch.int32, device=DEV)
    table = torch.empty(0, 4, dtype=torch.int32, device=DEV)
    assert ops.sdpa_decode_paged(rows(4), pool.dk, pool.dv, table, none).shape == (0, 512)
    ops.kv_append_paged(rows(2), rows(2), pool.dk, pool.dv, table, none)
    ops.kv_append_paged(rows(2), rows(2), pool.dk, pool.dv, pool.dtable, _dev(np.zeros(1, np.int32)),
                        cu_seqlens=_dev(np.zeros(2, np.int32)))
    assert ops.sdpa_prefill_packed_bf16(rows(4), rows(2), rows(2), _dev(np.zeros(3, np.int32)), 4, 2).shape == (0, 512)
    torch.cuda.synchronize()


def test_prefill_bad_offsets_are_cut_and_reported():
    """Offsets that fall, or leave the rows: nothing outside the rows is touched, and NMI_ERR_ASYNC."""
    rng = np.random.default_rng(33)
    q, k, v = _dev(_rand_bits(rng, 50, 4 * 128)), _dev(_rand_bits(rng, 50, 128)), _dev(_rand_bits(rng, 50, 128))
    for cu in ([0, 20, 51], [-1, 20, 50], [0, 30, 20], [2 ** 31 - 1, 2 ** 31 - 1, 2 ** 31 - 1], [-5, -5, -5]):
        announce("packed_bad", cu)
        out = torch.full((52, 4 * 128), 3.0, dtype=torch.bfloat16, device=DEV)
        ops.sdpa_prefill_packed_bf16(q, k, v, _dev(np.array(cu, np.int32)), 4, 1, out=out[1:51])
        torch.cuda.synchronize()
        assert (out[0] == 3).all() and (out[51] == 3).all()
        assert _lib.lib().nmi_async_status() == _lib.NMI_ERR_ASYNC
        assert _lib.lib().nmi_async_status() == 0


# --- together --------------------------------------------------------------------------------------


@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
def test_prompts_then_steps(kind):
    """Three conversations as a server runs them: the prompts appended and attended, then steps of one
    token each, appended and attended; every output against the oracle fed with the true cache."""
    announce("serve", kind)
    rng = np.random.default_rng(40)
    H, n_kv, page, lens, steps = 10, 2, 16, [37, 5, 64], 4
    f = (10000.0 ** (-np.arange(32) / 32)).astype(np.float32)
    pool = Pool(rng, [0, 0, 0], n_kv, page, kind, hold=[n + steps for n in lens])
    df, cu = _dev(f), np.concatenate([[0], np.cumsum(lens)]).astype(np.int32)

    def project(T):
        buf = _rand_bits(rng, T, (H + 2 * n_kv) * 128)
        d = _dev(buf)
        return d[:, :H * 128], d[:, H * 128:(H + n_kv) * 128], d[:, (H + n_kv) * 128:]

    q, k, v = project(sum(lens))
    start = torch.zeros(3, dtype=torch.int32, device=DEV)
    q, k = ops.kv_append_paged(k, v, pool.dk, pool.dv, pool.dtable, start, cu_seqlens=_dev(cu), q=q, inv_freq=df,
                               k_scale=pool.dks, v_scale=pool.dvs, q_out=q, k_out=k)
    o = ops.sdpa_prefill_packed_bf16(q, k, v, _dev(cu), H, n_kv)
    T = sum(lens)
    want = paged.prefill(*(_f64(bits(x.contiguous())).reshape(T, -1, 128) for x in (q, k, v)), cu)
    assert_parity(bits(o).reshape(want.shape), block.bf16_round_exact(want), "prompts")
    pos = _dev(np.array(lens, np.int32))
    for step in range(steps):
        q, k, v = project(3)
        q, _ = ops.kv_append_paged(k, v, pool.dk, pool.dv, pool.dtable, pos, q=q, inv_freq=df, k_scale=pool.dks,
                                   v_scale=pool.dvs)
        pos += 1
        o = ops.sdpa_decode_paged(q, pool.dk, pool.dv, pool.dtable, pos, k_scale=pool.dks, v_scale=pool.dvs)
        pool.k, pool.v = pool.host(pool.dk), pool.host(pool.dv)
        K, V = pool.values()
        want = paged.decode(_f64(bits(q)).reshape(3, H, 128), K, V, pool.table, [n + step + 1 for n in lens])
        assert_parity(bits(o).reshape(want.shape), block.bf16_round_exact(want), f"step {step}")
    assert _lib.lib().nmi_async_status() == 0


def test_a_captured_step_follows_the_sequences():
    """One graph of append and attention, replayed as the sequences grow (positions and page table are
    device data), with eager work between the replays: every replay gives the eager bytes."""
    announce("serve_graph")
    rng = np.random.default_rng(41)
    H, n_kv, page = 16, 4, 16
    starts = [30, 0, 700, -1]
    a, b = (Pool(np.random.default_rng(42), [max(0, s) for s in starts], n_kv, page, "bf16",
                 hold=[max(0, s) + 300 for s in starts]) for _ in range(2))
    f = _dev(np.ones(64, np.float32))
    sq, sk, sv = (_dev(_rand_bits(rng, 4, n * 128)) for n in (H, n_kv, n_kv))
    pos, lens = _dev(np.array(starts, np.int32)), _dev(np.array(starts, np.int32))
    out = torch.zeros(4, H * 128, dtype=torch.bfloat16, device=DEV)

    def step(pool, out):
        torch.add(pos, 1, out=lens)
        q, _ = ops.kv_append_paged(sk, sv, pool.dk, pool.dv, pool.dtable, pos, q=sq, inv_freq=f)
        ops.sdpa_decode_paged(q, pool.dk, pool.dv, pool.dtable, lens, out=out)

    eager = torch.zeros_like(out)
    step(b, eager)                                          # (writes position 30, 0, 700: the first replay's too)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=torch.cuda.Stream()):
        step(a, out)
    grow = torch.tensor([1, 1, 1, 0], dtype=torch.int32, device=DEV)
    for i in range(6):
        sk.copy_(_dev(_rand_bits(rng, 4, n_kv * 128)))
        sq.copy_(_dev(_rand_bits(rng, 4, H * 128)))
        out.zero_()
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        step(b, eager)
        torch.cuda.synchronize()
        assert torch.equal(out.view(torch.int16), eager.view(torch.int16)), i
        assert torch.equal(a.dk.view(torch.int16), b.dk.view(torch.int16))
        assert not out[3].any() and out[:3].abs().sum(-1).min() > 0
        pos += grow
    assert _lib.lib().nmi_async_status() == 0


def test_a_graph_may_hold_the_first_call():
    """The library's first paged call of a process inside a capture (its error word is allocated then)."""
    announce("first_call_captured")
    import subprocess
    import sys

    from tests.conftest import ROOT
    code = """
import torch
from nemotron_infer_amd import ops
q = torch.ones(1, 512, dtype=torch.bfloat16, device="cuda"); k = torch.ones(1, 128, dtype=torch.bfloat16, device="cuda")
pages = [torch.zeros(1, 1, 16, 128, dtype=torch.bfloat16, device="cuda") for _ in range(2)]
table = torch.zeros(1, 1, dtype=torch.int32, device="cuda"); pos = torch.zeros(1, dtype=torch.int32, device="cuda")
lens = torch.ones(1, dtype=torch.int32, device="cuda"); out = torch.zeros(1, 512, dtype=torch.bfloat16, device="cuda")
torch.cuda.synchronize()
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    ops.kv_append_paged(k, k, *pages, table, pos)
    ops.sdpa_decode_paged(q, *pages, table, lens, out=out)
for _ in range(3):
    out.zero_(); g.replay(); torch.cuda.synchronize()
    assert (out == 1).all()
"""
    r = subprocess.run([sys.executable, "-c", code], cwd=ROOT, capture_output=True, text=True, timeout=100)
    assert r.returncode == 0, r.stderr[-2000:]


def test_two_streams_and_two_threads():
    announce("paged_streams")
    rng = np.random.default_rng(50)
    pools = [Pool(rng, [900, 40 + i], 8, 16, "bf16") for i in range(2)]
    qs = [_dev(_rand_bits(rng, 2, 40 * 128)) for _ in range(2)]
    want = [p.decode(q) for p, q in zip(pools, qs)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(10):
        got = []
        for s, p, q in zip(streams, pools, qs):
            with torch.cuda.stream(s):
                got.append(p.decode(q))
        torch.cuda.synchronize()
        assert all(torch.equal(a.view(torch.int16), b.view(torch.int16)) for a, b in zip(got, want))
    results = [[], []]

    def work(i):
        with torch.cuda.stream(streams[0]):
            for _ in range(20):
                results[i].append(pools[i].decode(qs[i]))

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    for i in range(2):
        assert len(results[i]) == 20
        assert all(torch.equal(o.view(torch.int16), want[i].view(torch.int16)) for o in results[i])


def test_the_front_end_keeps_nothing():
    """References and device memory after many calls as before them; an error of the library is its
    exception, after which the next call runs."""
    announce("paged_front")
    pool = Pool(np.random.default_rng(51), [40, 7], 2, 16, "e4m3")
    q, k, pos = _dev(_rand_bits(np.random.default_rng(52), 2, 512)), torch.zeros(2, 256, dtype=torch.bfloat16, device=DEV), _dev(
        np.array([3, 4], np.int32))
    f, cu = _dev(np.ones(64, np.float32)), _dev(np.array([0, 1, 2], np.int32))

    def all_three():
        a, none = ops.kv_append_paged(k, k, pool.dk, pool.dv, pool.dtable, pos, q=q, inv_freq=f, k_scale=pool.dks, v_scale=pool.dvs)
        b = ops.sdpa_prefill_packed_bf16(a, k, k, cu, 4, 2)
        c = pool.decode(a)
        assert none is None and sys.getrefcount(a) == sys.getrefcount(b) == sys.getrefcount(c) == 2
        same = ops.sdpa_decode_paged(q, pool.dk, pool.dv, pool.dtable, pos, k_scale=pool.dks, v_scale=pool.dvs, out=c)
        assert same is c
        return c

    want = all_three()
    torch.cuda.synchronize()
    held = [q, k, pos, f, cu, pool.dk, pool.dv, pool.dtable, pool.dks, pool.dvs]
    counts, memory = [sys.getrefcount(x) for x in held], torch.cuda.memory_allocated()
    nones = sys.getrefcount(None)
    for _ in range(300):
        all_three()
    torch.cuda.synchronize()
    assert [sys.getrefcount(x) for x in held] == counts and torch.cuda.memory_allocated() == memory
    assert abs(sys.getrefcount(None) - nones) < 100
    small = torch.zeros(4, 2, 8, 128, dtype=torch.bfloat16, device=DEV)
    for _ in range(3):
        with pytest.raises(_lib.NmiError, match="page_size=8"):
            ops.sdpa_decode_paged(q, small, small, pool.dtable, pos)
        with pytest.raises(_lib.NmiError, match="page_size=8"):
            ops.kv_append_paged(k, k, small, small, pool.dtable, pos)
        with pytest.raises(_lib.NmiError, match="scale"):
            ops.sdpa_prefill_packed_bf16(q, k, k, cu, 4, 2, scale=-1.0)
    assert [sys.getrefcount(x) for x in held] == counts
    assert torch.equal(all_three().view(torch.int16), want.view(torch.int16))
