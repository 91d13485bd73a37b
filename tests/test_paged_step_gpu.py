"""GPU parity of a serving step on a paged cache: pages handed out on the device, keys and values under scales of
blocks of 16 positions, attention over them, key bounds of pages, attention of selected pages.

Bars (derived before the first run):
* whole numbers (tables, stacks, slots, lengths, selected places): equal.  Scores are summed in 64 bits and rounded
  to float32 on both sides: they differ only where a sum lies within 2^-50 of the middle of two floats.
* stored without rotation: scales and codes bit for bit (powers of two: one rounding of an exact quotient).
* rotated keys: the scale is a power of two and equal unless a value lies within the rotation's error of a border;
  codes between the rounded ends of [exact - d, exact + d] / scale, d = (|x| + |y|) 2^-22: a float32 sine and cosine off
  by 2^-24 of their value and half a turn's 2^-30, 2^-23 together on both terms, and one rounding of 2^-24.
* k_out and q_out: as test_paged_gpu.py's.
* attention: the parity gate of oracle.linear.parity against float64 rounded once, as test_paged_gpu.py's; scales
  of blocks add one rounding of 2^-24 to a score and one to a weight.
* bounds: the smallest and largest of float32 values, rounded once: equal (codes times powers of two are exact; times
  other scales the product is rounded to float32 first on both sides).
"""
import sys
import threading

import numpy as np
import pytest
import torch

from nemotron_infer_amd import _lib, ops
from oracle import block, e4m3, paged
from tests.gpu_util import DEV, announce, assert_parity, bits
from tests.test_paged_edges_gpu import BAD_OFFSETS
from tests.test_paged_gpu import LUT, NAN_BF16, Pool, _between, _bf16, _dev, _f64, _rand_bits

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _no_pending_error():
    _lib.lib().nmi_async_status()
    yield
    torch.cuda.synchronize()
    _lib.lib().nmi_async_status()


class BlockPool(Pool):
    """A pool of e4m3 pages under scales [n_pages, n_kv, page / 16]: powers of two from 2^-12 to 2^-1 (powers: any up
    to 1).  What lies behind a sequence's length is NaN, scales of blocks of nobody too."""

    def __init__(self, rng, lens, n_kv, page, kind="block", powers=True, **kw):
        super().__init__(rng, lens, n_kv, page, "e4m3", **kw)
        shape = (self.k.shape[0], n_kv, page // 16)
        self.kind, self.powers = kind, powers
        self.ks, self.vs = np.full(shape, np.nan, np.float32), np.full(shape, np.nan, np.float32)
        for b, n in enumerate(self.lens):
            for p0 in range(0, max(0, int(n)), 16):
                for s in (self.ks, self.vs):
                    made = 2.0 ** rng.integers(-12, 0, n_kv) if powers else rng.uniform(1e-3, 0.05, n_kv)
                    s[self.table[b, p0 // page], :, p0 % page // 16] = made
        self.dks, self.dvs = _dev(self.ks), _dev(self.vs)

    def values(self):
        spread = lambda s: np.repeat(s.astype(np.float64), 16, axis=2)[..., None]  # noqa: E731
        return LUT[self.k] * spread(self.ks), LUT[self.v] * spread(self.vs)

    def host(self, t):
        return t.contiguous().view(torch.uint8).cpu().numpy()

    def fetch(self):
        """The host's copy as the GPU's."""
        self.k, self.v = self.host(self.dk), self.host(self.dv)
        self.ks, self.vs = self.dks.cpu().numpy(), self.dvs.cpu().numpy()


def _pool(kind, rng, lens, n_kv, page, **kw):
    return (BlockPool if kind == "block" else Pool)(rng, lens, n_kv, page, kind, **kw)


def _check_decode(rng, lens, H, n_kv, page, qscale=0.3, label="", **kw):
    pool = BlockPool(rng, lens, n_kv, page, **kw)
    q = _rand_bits(rng, len(lens), H * 128, scale=qscale)
    o = pool.decode(_dev(q))
    torch.cuda.synchronize()
    want = paged.decode(_f64(q).reshape(len(lens), H, 128), *pool.values(), pool.table, pool.lens)
    got = bits(o).reshape(want.shape)
    live = pool.lens > 0
    assert not got[~live].any()
    if live.any():
        assert_parity(got[live], block.bf16_round_exact(want[live]), label, per_row_scales=True)
    assert _lib.lib().nmi_async_status() == 0


# --- attention under scales of blocks --------------------------------------------------------------


@pytest.mark.parametrize("n", [0, 1, 2, 15, 16, 17, 31, 32, 33, 47, 48, 49, 64, 65, 129, 777, 1025])
def test_decode_lengths(n):
    announce("block_decode", n)
    _check_decode(np.random.default_rng(n), [n], 40, 8, 16, label=f"{n}")


@pytest.mark.parametrize("H,n_kv", [(1, 1), (8, 8), (7, 1), (17, 1), (40, 1), (66, 2)])
def test_decode_head_groups(H, n_kv):
    announce("block_heads", H, n_kv)
    _check_decode(np.random.default_rng(H), [45, 0, 300, 1], H, n_kv, 32, label=f"{H}/{n_kv}")


@pytest.mark.parametrize("page", [16, 32, 64, 1024])
@pytest.mark.parametrize("layout", ["heads", "tokens", "slice"])
def test_decode_pages_and_layouts(page, layout):
    announce("block_layout", page, layout)
    _check_decode(np.random.default_rng(page), [70, 513, 16, 1300], 16, 4, page, label=f"{page} {layout}", layout=layout)


def test_decode_any_positive_scales_and_ragged_batches():
    rng = np.random.default_rng(7)
    announce("block_scales")
    _check_decode(rng, [300, 33, 1], 8, 2, 32, powers=False, label="scales that are no powers of two")
    for lens in ([int(n) for n in rng.integers(-3, 60, 150)], [3] * 70 + [5000] + [17] * 60, [20000, 33], [0] * 3):
        announce("block_ragged", len(lens), max(lens))
        _check_decode(rng, lens, 8, 2, 16, label=f"{len(lens)} sequences")


@pytest.mark.parametrize("batch,H,n_kv,page,width", [(3, 40, 8, 16, 40), (3, 40, 8, 16, 41), (40, 16, 8, 64, 16), (40, 16, 8, 64, 17), (70, 33, 1, 32, 32),
                                                     (300, 4, 1, 256, 4)])
def test_decode_on_both_sides_of_the_launches_choice(batch, H, n_kv, page, width):
    """Tables whose rows hold just so many positions as a workgroup takes alone, and more; lengths of all kinds in them."""
    announce("block_whole", batch, H, n_kv, page * width)
    rng = np.random.default_rng(batch + width)
    lens = [int(n) for n in rng.integers(0, page * width + 1, batch)]
    lens[0], lens[-1], lens[1] = page * width, 1, 0
    _check_decode(rng, lens, H, n_kv, page, label=f"{page * width}", width=width)


def test_decode_is_the_same_every_time_and_equals_scales_of_heads():
    """One scale everywhere: as under a scale per head, up to where float32 rounds (powers of two: nowhere)."""
    announce("block_repeat")
    rng = np.random.default_rng(11)
    pool = Pool(rng, [3000, 17, 900], 8, 64, "e4m3")
    pool.dks.fill_(2.0 ** -6), pool.dvs.fill_(2.0 ** -5)
    q = _dev(_rand_bits(rng, 3, 40 * 128))
    whole = pool.decode(q)
    shape = (pool.k.shape[0], 8, 4)
    pool.dks, pool.dvs = torch.full(shape, 2.0 ** -6, device=DEV), torch.full(shape, 2.0 ** -5, device=DEV)
    first = pool.decode(q)
    assert_parity(bits(first), bits(whole), "scales of heads")
    for _ in range(5):
        assert torch.equal(pool.decode(q).view(torch.int16), first.view(torch.int16))


@pytest.mark.parametrize("k_power,v_power", [(-100, -90), (100, 90), (-20, 100), (20, -100)])
def test_decode_of_far_magnitudes(k_power, v_power):
    """Keys and values of any magnitude that their scales can say, within what the header allows."""
    announce("block_far_scales", k_power, v_power)
    rng = np.random.default_rng(14)
    pool = BlockPool(rng, [200, 31], 2, 16)
    pool.ks, pool.vs = pool.ks * np.float32(2.0 ** (k_power + 6)), pool.vs * np.float32(2.0 ** (v_power + 6))
    pool.dks, pool.dvs = _dev(pool.ks), _dev(pool.vs)
    q = _rand_bits(rng, 2, 8 * 128, scale=2.0 ** -k_power if k_power < 100 else 2.0 ** -106)
    o = pool.decode(_dev(q))
    want = paged.decode(_f64(q).reshape(2, 8, 128), *pool.values(), pool.table, pool.lens)
    assert_parity(bits(o).reshape(want.shape), block.bf16_round_exact(want), "far", per_row_scales=True)


def test_decode_nan_codes_bad_pages_and_lengths():
    """A NaN in v stays in its dim and head; a bad page or length makes its sequence NaN and is reported once."""
    announce("block_bad")
    rng = np.random.default_rng(13)
    pool = BlockPool(rng, [90, 200, 40], 2, 32)
    q = _rand_bits(rng, 3, 8 * 128, scale=0.3)
    good = bits(pool.decode(_dev(q))).reshape(3, 8, 128)
    pool.v[pool.table[1, 2], 1, 5, 77] = 0x7F
    pool.dv = pool._to_dev(pool.v)
    got = bits(pool.decode(_dev(q))).reshape(3, 8, 128)
    torch.cuda.synchronize()
    at = np.zeros(got.shape, bool)
    at[1, 4:, 77] = True
    assert np.isnan(_f64(got[at])).all() and np.array_equal(got[~at], good[~at])
    for change in ("page", "negative", "length"):
        lens, table = pool.lens.copy(), pool.table.copy()
        if change == "length":
            lens[1] = table.shape[1] * 32 + 1
        else:
            table[1, 3] = pool.k.shape[0] if change == "page" else -1
        pool.dtable = _dev(table)
        got = bits(pool.decode(_dev(q), lens=lens)).reshape(3, 8, 128)
        torch.cuda.synchronize()
        assert np.isnan(_f64(got[1])).all()
        # (another length deals the tiles of all sequences to other waves: their float32 sums go in another order, so that
        # two right results differ as each may from the exact one)
        if change == "length":
            assert_parity(got[[0, 2]], good[[0, 2]], change)
        else:
            assert np.array_equal(got[[0, 2]], good[[0, 2]])
        assert _lib.lib().nmi_async_status() == _lib.NMI_ERR_ASYNC and _lib.lib().nmi_async_status() == 0


# --- append under scales of blocks -----------------------------------------------------------------


def _check_append(rng, starts, lens, H, n_kv, page, rotary, interleaved, layout="heads", lead=0, tail=0, packed=True, in_place=False,
                  grow=0.0, x=None, powers=True, held=None):
    """held: positions that the pool holds of each sequence (default: all before its new ones)."""
    starts = np.array(starts, np.int32)
    T = lead + sum(lens) + tail
    cu = lead + np.concatenate([[0], np.cumsum(lens)]).astype(np.int32)
    hold = [max(0, int(s)) + n for s, n in zip(starts, lens)]
    pool = BlockPool(rng, [max(0, int(s)) for s in starts], n_kv, page, layout=layout, hold=hold, powers=powers)
    buf = _rand_bits(rng, T, (H + 2 * n_kv) * 128)
    if grow:
        buf = block.bf16_round_exact(_f64(buf) * np.exp2(rng.uniform(-grow, grow, (T, H + 2 * n_kv))).repeat(128, axis=1))
    cols = [0, H * 128, (H + n_kv) * 128, (H + 2 * n_kv) * 128]
    if x is not None:
        buf[:, cols[1]:] = x
    dbuf = _dev(buf)
    dq, dk, dv = (dbuf[:, a:b] for a, b in zip(cols, cols[1:]))
    q, k, v = (_f64(buf[:, a:b]).reshape(T, -1, 128) for a, b in zip(cols, cols[1:]))
    f = (10000.0 ** (-np.arange(rotary // 2) / (rotary // 2))).astype(np.float32) if rotary else None
    qo = (dq if in_place else torch.full((T, H * 128), 5.0, dtype=torch.bfloat16, device=DEV)) if rotary else None
    ko = (dk if in_place else torch.full((T, n_kv * 128), 5.0, dtype=torch.bfloat16, device=DEV)) if rotary else None
    pool.fetch()
    old = [pool.k.copy(), pool.v.copy(), pool.ks.copy(), pool.vs.copy()]
    ops.kv_append_paged(dk, dv, pool.dk, pool.dv, pool.dtable, _dev(starts), cu_seqlens=_dev(cu) if packed else None,
                        q=dq if rotary else None, inv_freq=None if f is None else _dev(f), interleaved=interleaved,
                        k_scale=pool.dks, v_scale=pool.dvs, q_out=qo, k_out=ko)
    torch.cuda.synchronize()
    assert _lib.lib().nmi_async_status() == 0
    rows = paged.positions(T, starts, cu if packed else None)
    pool.fetch()
    if not rows:
        assert all(np.array_equal(a, b, equal_nan=True) for a, b in zip(old, (pool.k, pool.v, pool.ks, pool.vs)))
        return
    r, seq, pos = (np.array(c) for c in zip(*rows))
    slack, none = np.zeros_like(k), np.zeros_like(v)
    if rotary:
        slack[r] = paged.partner_sum(k[r], rotary, interleaved) * 2.0 ** -22
        k[r], q[r] = (paged.rotate(y[r], pos.astype(np.float64), f, interleaved) for y in (k, q))
        pq = paged.partner_sum(_f64(buf[:, :cols[1]]).reshape(T, -1, 128)[r], rotary, interleaved) * 2.0 ** -20
        for out, exact, d, src in ((qo, q[r], pq, buf[:, :cols[1]]), (ko, k[r], 4 * slack[r], buf[:, cols[1]:cols[2]])):
            host = bits(out)
            _between(_f64(host[r]).reshape(exact.shape), exact, d, _bf16)
            rest = np.setdiff1d(np.arange(T), r)
            assert np.array_equal(host[rest], src[rest] if in_place else np.full_like(src[rest], 0x40A0))
    at = (pool.table[seq, pos // page], slice(None), pos % page)
    for name, codes, scales, was, was_scale, y, d in (("k", pool.k, pool.ks, old[0], old[2], k, slack),
                                                       ("v", pool.v, pool.vs, old[1], old[3], v, none)):
        want, want_scale = LUT[was].copy(), was_scale.astype(np.float64)
        paged.append_blocks(want, want_scale, y, rows, pool.table, page)
        assert np.array_equal(scales.astype(np.float64), want_scale, equal_nan=True), name
        new = np.zeros(codes.shape, bool)
        new[at] = True
        # codes moved to a new scale, and all others that are not new: exactly
        assert np.array_equal(LUT[codes[~new]], want[~new], equal_nan=True), name
        stay = ~new & (LUT[was] == want)
        assert np.array_equal(codes[stay], was[stay]), name
        s = want_scale[pool.table[seq, pos // page], :, pos % page // 16][..., None]
        if np.isfinite(y[r]).all():
            _between(LUT[codes[at]], y[r] / s, d[r] / s, paged.round_e4m3)
        else:
            assert np.array_equal(LUT[codes[at]], want[at], equal_nan=True)


@pytest.mark.parametrize("rotary,interleaved", [(0, False), (128, False), (128, True), (64, False), (16, True), (112, False), (96, True)])
def test_append_prompts(rotary, interleaved):
    announce("block_append", rotary, interleaved)
    rng = np.random.default_rng(rotary)
    _check_append(rng, [0, 5, 31, 0, 100], [70, 1, 33, 0, 16], 8, 2, 32, rotary, interleaved, grow=4)
    _check_append(rng, [7, 0, 15, 14], [20, 3, 2, 18], 5, 5, 16, rotary, interleaved, layout="tokens", lead=2, tail=3)
    _check_append(rng, [9, 0], [300, 40], 40, 8, 128, rotary, interleaved, layout="slice", in_place=True)


@pytest.mark.parametrize("rotary", [0, 128])
@pytest.mark.parametrize("batch", [1, 3, 64, 65, 200, 1100])
def test_append_one_token_each(batch, rotary):
    announce("block_append_decode", batch, rotary)
    rng = np.random.default_rng(batch)
    starts = rng.integers(0, 300 if batch < 200 else 40, batch)
    starts[batch // 2] = -1 if batch > 1 else 40
    for packed in (False, True):
        _check_append(rng, starts, [1] * batch, 6, 2, 16 if batch < 100 else 64, rotary, False, packed=packed, in_place=not packed,
                      grow=6)


def test_append_many_sequences_of_odd_lengths():
    announce("block_append_many")
    rng = np.random.default_rng(20)
    lens = [int(n) for n in rng.integers(0, 5, 300)]
    _check_append(rng, [int(s) for s in rng.integers(-2, 40, 300)], lens, 4, 1, 16, 32, True, lead=1, tail=70, grow=4)
    _check_append(rng, [15] * 130, [18] * 130, 2, 2, 32, 0, False)              # the most blocks that rows can need


@pytest.mark.parametrize("packed", [False, True])
def test_append_rotates_keys_alone(packed):
    """No q, and no k returned: the cache as with them."""
    announce("block_append_keys", packed)
    rng = np.random.default_rng(28)
    a, b = (BlockPool(np.random.default_rng(29), [3, 20, 7], 2, 32, hold=[40, 40, 40]) for _ in range(2))
    x, f, start = _dev(_rand_bits(rng, 3, 8 * 128)), _dev(np.ones(64, np.float32)), _dev(np.array([3, 20, 7], np.int32))
    k, v, q = x[:, :256], x[:, 256:512], x[:, 512:]
    cu = _dev(np.arange(4, dtype=np.int32)) if packed else None
    got = ops.kv_append_paged(k, v, a.dk, a.dv, a.dtable, start, cu_seqlens=cu, inv_freq=f, k_scale=a.dks, v_scale=a.dvs)
    ops.kv_append_paged(k, v, b.dk, b.dv, b.dtable, start, cu_seqlens=cu, q=q, inv_freq=f, k_scale=b.dks, v_scale=b.dvs,
                        k_out=torch.empty_like(k))
    assert got == (None, None)
    for s, t in ((a.dk, b.dk), (a.dv, b.dv), (a.dks, b.dks), (a.dvs, b.dvs)):
        assert _same(s, t)


def test_the_largest_page():
    """Pages of 2^20 positions: appended across a block border, bounded, and attended."""
    announce("block_largest_page")
    rng = np.random.default_rng(30)
    page, n = 1 << 20, 40
    pages = [torch.zeros(2, 1, page, 128, dtype=torch.uint8, device=DEV) for _ in range(2)]
    scales = [torch.ones(2, 1, page // 16, device=DEV) for _ in range(2)]
    table, start = _dev(np.array([[1, 0]], np.int32)), page - 30
    k, v, q = (_rand_bits(rng, m, 128) for m in (n, n, 1))
    args = dict(cu_seqlens=_dev(np.array([0, n], np.int32)), k_scale=scales[0], v_scale=scales[1])
    ops.kv_append_paged(_dev(k), _dev(v), *pages, table, _dev(np.array([start], np.int32)), **args)
    bounds = torch.zeros(2, 1, 2, 128, dtype=torch.bfloat16, device=DEV)
    ops.kv_bounds_paged(pages[0], table, _dev(np.array([start], np.int32)), bounds, cu_seqlens=args["cu_seqlens"], tokens=n, k_scale=scales[0])
    lens = _dev(np.array([start + n], np.int32))
    o = ops.sdpa_decode_paged(_dev(q), *pages, table, lens, k_scale=scales[0], v_scale=scales[1], scale=2.0)
    sparse = ops.sdpa_decode_paged_sparse(_dev(q), *pages, table, lens, bounds, 1, k_scale=scales[0], v_scale=scales[1], scale=2.0)
    torch.cuda.synchronize()
    held = []                                             # the new positions' values, and the zeros before them
    for c, s, x in zip(pages, scales, (k, v)):
        rows = torch.cat([c[1, 0, -30:], c[0, 0, :10]]).cpu().numpy()
        by = torch.cat([s[1, 0].repeat_interleave(16)[-30:], s[0, 0, :1].repeat(10)]).cpu().numpy()
        held.append(LUT[rows] * by[:, None])
        assert np.abs(held[-1] - _f64(x)).max() <= 2.0 ** -4 * np.abs(_f64(x)).max()
    e = np.concatenate([np.zeros(start), 2.0 * (held[0] @ _f64(q)[0])])
    w = np.exp(e - e.max())
    assert_parity(bits(o), block.bf16_round_exact((w[start:] @ held[1])[None] / w.sum()), "largest page")
    w = np.exp(e[page:] - e[page:].max())
    assert_parity(bits(sparse), block.bf16_round_exact((w @ held[1][30:])[None] / w.sum()), "its newest page")
    whole = np.concatenate([np.zeros((1, 128)), held[0][:30]])
    assert np.array_equal(_f64(bits(bounds[1, 0])), np.stack([_bf16(whole.min(0)), _bf16(whole.max(0))]))
    assert not bounds[0].any() and _lib.lib().nmi_async_status() == 0


def test_append_token_by_token_follows_the_values():
    """Blocks that fill as magnitudes grow, fall and vanish: each step's scales, moved codes and new ones."""
    announce("block_append_growth")
    rng = np.random.default_rng(25)
    pool, batch, n_kv, page = BlockPool(rng, [0, 0, 0], 2, 32, hold=[70] * 3), 3, 2, 32
    starts = np.array([0, 5, 30], np.int32)
    values, scales = [LUT[pool.k].copy(), LUT[pool.v].copy()], [pool.ks.astype(np.float64), pool.vs.astype(np.float64)]
    pool.dks[:], pool.dvs[:] = 2.0 ** -20, 2.0 ** -20
    pool.dk.zero_(), pool.dv.zero_()
    for i in range(2):
        values[i][:], scales[i][:] = 0.0, 2.0 ** -20
    for step in range(40):
        size = 2.0 ** rng.integers(-30, 30, (batch, 2 * n_kv, 1)) if step % 3 else np.zeros((batch, 2 * n_kv, 1))
        x = block.bf16_round_exact(rng.standard_normal((batch, 2 * n_kv, 128)) * size)
        d = _dev(x.reshape(batch, -1))
        ops.kv_append_paged(d[:, :256], d[:, 256:], pool.dk, pool.dv, pool.dtable, _dev(starts), k_scale=pool.dks, v_scale=pool.dvs)
        pool.fetch()
        for i, (codes, s) in enumerate(((pool.k, pool.ks), (pool.v, pool.vs))):
            rows = [(b, b, int(starts[b])) for b in range(batch)]
            paged.append_blocks(values[i], scales[i], _f64(x)[:, i * n_kv:(i + 1) * n_kv], rows, pool.table, page)
            assert np.array_equal(s.astype(np.float64), scales[i]) and np.array_equal(LUT[codes], values[i]), step
        starts += 1
    assert len(np.unique(pool.ks)) > 8


def test_append_values_at_the_ends_of_float32():
    """Zeros, the smallest and largest values, borders of scales, NaN and infinities, in prompts and by token."""
    announce("block_append_edges")
    rng = np.random.default_rng(26)
    vals = [0.0, 2.0 ** -133, 2.0 ** -126, 2.0 ** -117, 2.0 ** -120, 1.0, 1.75, 1.7578125, 448.0, 450.0, 3.3895e38, 1.75 * 2.0 ** 127, -2.0 ** 127]
    for T, packed in ((18, True), (5, False)):
        x = np.zeros((T, 2 * 2 * 128))
        for t in range(T):
            for h in range(4):
                x[t, h * 128:h * 128 + 3] = rng.choice(vals, 3) if t % 4 else 0.0
        xb = block.bf16_round_exact(x)
        _check_append(rng, [0] if packed else [0, 3, 7, 15, 16], [T] if packed else [1] * T, 2, 2, 16, 0, False, x=xb, packed=packed)
        for bad in (NAN_BF16, 0x7F80, 0xFF80):
            xb[T // 2, 5::128] = bad
            xb[T - 1, 7] = bad
        _check_append(rng, [0] if packed else [0, 3, 7, 15, 16], [T] if packed else [1] * T, 2, 2, 16, 0, False, x=xb, packed=packed)


def test_append_under_scales_that_are_no_powers_of_two():
    """They count as the next power of two, and the block's codes move with them."""
    announce("block_append_other_scales")
    rng = np.random.default_rng(27)
    _check_append(rng, [5, 16, 37, 12], [1] * 4, 4, 2, 16, 0, False, packed=False, powers=False)
    _check_append(rng, [5, 16, 37, 12], [3, 20, 2, 9], 4, 2, 32, 64, False, powers=False)


def test_append_bad_places_are_skipped_and_reported():
    rng = np.random.default_rng(22)
    f = _dev(np.ones(8, np.float32))
    for packed in (False, True):
        for table, starts in (([[0], [-1], [1]], [3, 4, 5]), ([[0], [2], [1]], [3, 4, 5]), ([[0], [0], [1]], [3, 16, 5]),
                              ([[0], [0], [1]], [3, 2 ** 31 - 1, 5])):
            announce("block_append_bad", packed, table, starts)
            pages = [torch.zeros(2, 1, 16, 128, dtype=torch.float8_e4m3fn, device=DEV) for _ in range(2)]
            scales = [torch.full((2, 1, 1), 2.0 ** -9, device=DEV) for _ in range(2)]
            k, v, q = (_dev(_rand_bits(rng, 3, 128)) for _ in range(3))
            q_out, _ = ops.kv_append_paged(k, v, *pages, _dev(np.array(table, np.int32)), _dev(np.array(starts, np.int32)), q=q,
                                           inv_freq=f, k_scale=scales[0], v_scale=scales[1],
                                           cu_seqlens=_dev(np.arange(4, dtype=np.int32)) if packed else None)
            torch.cuda.synchronize()
            got = LUT[pages[1].view(torch.uint8).cpu().numpy()][:, 0] * scales[1].cpu().numpy().reshape(2, 1, 1)
            assert int((np.abs(got).sum(-1) > 0).sum()) == 2
            for page, place, row in ((0, 3, 0), (1, 5, 2)):
                assert np.allclose(got[page, place], _f64(bits(v[row])), rtol=2.0 ** -4, atol=2.0 ** -10 * float(scales[1][page, 0, 0]))
            assert q_out.abs().sum(-1).min() > 0
            assert _lib.lib().nmi_async_status() == _lib.NMI_ERR_ASYNC and _lib.lib().nmi_async_status() == 0


@pytest.mark.parametrize("T,cu", BAD_OFFSETS, ids=[str(i) for i in range(len(BAD_OFFSETS))])
def test_append_bad_offsets_are_cut_and_reported(T, cu):
    """Each row of the rows given is stored at most once, for a sequence that its offsets give it to and at its place
    there; a row behind which no earlier sequence ends is stored if one has it; all others stay."""
    announce("block_bad_offsets", T, cu[:8])
    rng = np.random.default_rng(T + len(cu))
    batch, page = len(cu) - 1, 16
    starts = rng.integers(0, 40, batch).astype(np.int32)
    spans = [(min(max(a, 0), T), max(min(max(a, 0), T), min(max(b, 0), T))) for a, b in zip(cu, cu[1:])]
    rows, end = [], 0
    for b, (x, y) in enumerate(spans):
        rows += [(t, b, int(starts[b]) + t - x) for t in range(max(x, end), y)]
        end = max(end, y if y > x else 0)
    pool = BlockPool(rng, [int(s) for s in starts], 1, page, hold=[int(s) + y - x for s, (x, y) in zip(starts, spans)])
    x = _rand_bits(rng, T, 256)
    d = _dev(x)
    pool.fetch()
    want = [(LUT[c].copy(), s.astype(np.float64)) for c, s in ((pool.k, pool.ks), (pool.v, pool.vs))]
    ops.kv_append_paged(d[:, :128], d[:, 128:], pool.dk, pool.dv, pool.dtable, _dev(starts), cu_seqlens=_dev(np.array(cu)),
                        k_scale=pool.dks, v_scale=pool.dvs)
    torch.cuda.synchronize()
    assert _lib.lib().nmi_async_status() == _lib.NMI_ERR_ASYNC and _lib.lib().nmi_async_status() == 0
    pool.fetch()
    for i, (codes, scales) in enumerate(((pool.k, pool.ks), (pool.v, pool.vs))):
        paged.append_blocks(*want[i], _f64(x)[:, 128 * i:128 * i + 128].reshape(T, 1, 128), rows, pool.table, page)
        assert np.array_equal(LUT[codes], want[i][0], equal_nan=True)
        assert np.array_equal(scales.astype(np.float64), want[i][1], equal_nan=True)


def test_append_and_decode_past_32_bits():
    """Pages whose bytes lie more than 2^32 from the pool's start, and scales behind them."""
    announce("block_large_pool")
    n_pages, n_kv, page = 140000, 8, 32
    k_pages = torch.empty(n_pages, n_kv, page, 128, dtype=torch.uint8, device=DEV)
    v_pages = torch.empty_like(k_pages)
    assert k_pages.numel() > 1 << 32
    scales = [torch.empty(n_pages, n_kv, 2, device=DEV) for _ in range(2)]
    rng = np.random.default_rng(24)
    k, v = (_rand_bits(rng, 60, n_kv * 128) for _ in range(2))
    table = np.array([[n_pages - 1, 133001], [131999, n_pages - 2]], np.int32)
    zeros = _dev(np.zeros(2, np.int32))
    ops.kv_append_paged(_dev(k), _dev(v), k_pages, v_pages, _dev(table), zeros, cu_seqlens=_dev(np.array([0, 40, 60], np.int32)),
                        k_scale=scales[0], v_scale=scales[1])
    q = _rand_bits(rng, 2, 16 * 128)
    o = ops.sdpa_decode_paged(_dev(q), k_pages, v_pages, _dev(table), _dev(np.array([40, 20], np.int32)), k_scale=scales[0],
                              v_scale=scales[1])
    bounds = torch.zeros(n_pages, n_kv, 2, 128, dtype=torch.bfloat16, device=DEV)
    ops.kv_bounds_paged(k_pages, _dev(table), zeros, bounds, cu_seqlens=_dev(np.array([0, 40, 60], np.int32)), tokens=60,
                        k_scale=scales[0])
    torch.cuda.synchronize()
    small = {int(t): i for i, t in enumerate(table.flat)}
    held = []
    for pages, s in ((k_pages, scales[0]), (v_pages, scales[1])):
        ids = torch.tensor(list(small), device=DEV)
        held.append(np.nan_to_num(LUT[pages[ids].cpu().numpy()] * np.repeat(s[ids].cpu().numpy(), 16, axis=2)[..., None]))
    local = np.vectorize(small.get)(table)
    want = paged.decode(_f64(q).reshape(2, 16, 128), *held, local, [40, 20])
    assert_parity(bits(o).reshape(want.shape), block.bf16_round_exact(want), "far")
    row = _f64(v[:16]).reshape(16, n_kv, 128)
    assert np.abs(held[1][0][:, :16].transpose(1, 0, 2) - row).max() <= 2.0 ** -4 * np.abs(row).max()
    assert np.array_equal(_f64(bits(bounds[n_pages - 1])), paged.page_bounds(held[0][:1])[0])
    assert not bounds[131999].any() and _lib.lib().nmi_async_status() == 0


# --- bounds ----------------------------------------------------------------------------------------


def _f32_keys(pool):
    """The keys that the pool holds, products rounded to float32."""
    if pool.kind == "bf16":
        return _f64(pool.k)
    s = pool.ks[:, None, None] if pool.kind == "e4m3" else np.repeat(pool.ks, 16, axis=2)[..., None]
    return (LUT[pool.k].astype(np.float32) * s).astype(np.float64)


@pytest.mark.parametrize("kind", ["bf16", "e4m3", "block"])
@pytest.mark.parametrize("page", [16, 32, 64, 256, 2048])
def test_bounds(kind, page):
    announce("bounds", kind, page)
    rng = np.random.default_rng(page)
    starts, lens = [0, page - 1, 5, page, 2 * page - 1, 3, -1], [page, 1, 3 * page, page - 1, 0, page - 4, 2 * page]
    pool = _pool(kind, rng, [max(0, s) + n for s, n in zip(starts, lens)], 3, page, layout="tokens" if page == 32 else "heads")
    pool.k[pool.table[2, 1], 1, 7, 9] = 0x7F if kind != "bf16" else NAN_BF16
    pool.dk = pool._to_dev(pool.k)
    cu = np.concatenate([[0], np.cumsum(lens)]).astype(np.int32)
    old = _rand_bits(rng, pool.k.shape[0], 3, 2, 128)
    bounds = _dev(old)
    got = ops.kv_bounds_paged(pool.dk, pool.dtable, _dev(np.array(starts, np.int32)), bounds, cu_seqlens=_dev(cu), tokens=int(cu[-1]),
                              k_scale=pool.dks)
    assert got is bounds
    want = old.copy()
    with np.errstate(invalid="ignore"):
        every = block.bf16_round_exact(paged.page_bounds(_f32_keys(pool)))
    done = [pool.table[b, j] for b, (s, n) in enumerate(zip(starts, lens)) if s >= 0 for j in range(s // page, (s + n) // page)]
    assert len(done) == 5
    want[done] = every[done]
    assert np.array_equal(_f64(bits(bounds)), _f64(want), equal_nan=True)
    assert np.isnan(_f64(bits(bounds)[pool.table[2, 1], 1, :, 9])).all()
    # one token each
    bounds.copy_(_dev(old))
    ends = np.array([page - 1, page - 1, 5, 2 * page - 1, 2 * page - 2, 3, -1], np.int32)
    ops.kv_bounds_paged(pool.dk, pool.dtable, _dev(ends), bounds, k_scale=pool.dks)
    want = old.copy()
    done = [pool.table[b, e // page] for b, e in enumerate(ends) if (e + 1) % page == 0 and e >= 0]
    assert len(done) == 3
    want[done] = every[done]
    assert np.array_equal(_f64(bits(bounds)), _f64(want), equal_nan=True) and _lib.lib().nmi_async_status() == 0


def test_bounds_of_many_sequences_and_bad_data():
    announce("bounds_many")
    rng = np.random.default_rng(61)
    lens = [int(n) for n in rng.integers(0, 50, 300)]
    starts = [int(s) for s in rng.integers(-2, 40, 300)]
    pool = BlockPool(rng, [max(0, s) + n for s, n in zip(starts, lens)], 1, 16)
    cu = np.concatenate([[0], np.cumsum(lens)]).astype(np.int32)
    bounds = torch.zeros(pool.k.shape[0], 1, 2, 128, dtype=torch.bfloat16, device=DEV)
    args = (pool.dk, pool.dtable, _dev(np.array(starts, np.int32)), bounds)
    ops.kv_bounds_paged(*args, cu_seqlens=_dev(cu), tokens=int(cu[-1]), k_scale=pool.dks)
    want = np.zeros((pool.k.shape[0], 1, 2, 128))
    with np.errstate(invalid="ignore"):
        every = _bf16(paged.page_bounds(_f32_keys(pool)))
    for b, (s, n) in enumerate(zip(starts, lens)):
        for j in range(s // 16, (s + n) // 16) if s >= 0 else ():
            want[pool.table[b, j]] = every[pool.table[b, j]]
    assert np.array_equal(_f64(bits(bounds)), want) and _lib.lib().nmi_async_status() == 0
    for table, cu in (([[pool.k.shape[0], 0]], [0, 16]), ([[-1, 0]], [0, 16]), ([[0, 1]], [0, 100]), ([[0, 1]], [-3, 16]), ([[0, 1]], [5, 2])):
        announce("bounds_bad", table, cu)
        before = bounds.clone()
        ops.kv_bounds_paged(pool.dk, _dev(np.array(table, np.int32)), _dev(np.zeros(1, np.int32)), bounds,
                            cu_seqlens=_dev(np.array(cu, np.int32)), tokens=40, k_scale=pool.dks)
        torch.cuda.synchronize()
        assert _lib.lib().nmi_async_status() == _lib.NMI_ERR_ASYNC and _lib.lib().nmi_async_status() == 0
        assert torch.equal(bounds[2:].view(torch.int16), before[2:].view(torch.int16))


# --- selected pages --------------------------------------------------------------------------------


def _check_sparse(rng, kind, lens, H, n_kv, page, select, bounds=None, qscale=0.3, scale=None, label="", **kw):
    pool = _pool(kind, rng, lens, n_kv, page, **kw)
    if bounds is None:
        with np.errstate(invalid="ignore"):
            bounds = block.bf16_round_exact(np.nan_to_num(paged.page_bounds(_f32_keys(pool)), nan=7.0))
    else:
        bounds = bounds(pool)
    B = len(lens)
    q = _rand_bits(rng, B, H * 128, scale=qscale)
    places = torch.full((B, n_kv, select), -7, dtype=torch.int32, device=DEV)
    kw = {} if scale is None else {"scale": scale}
    call = lambda **more: ops.sdpa_decode_paged_sparse(_dev(q), pool.dk, pool.dv, pool.dtable, _dev(pool.lens), _dev(bounds), select,  # noqa: E731
                                                       k_scale=pool.dks, v_scale=pool.dvs, **kw, **more)
    o = call(selected=places)
    torch.cuda.synchronize()
    assert _lib.lib().nmi_async_status() == 0
    x, edges = _f64(q).reshape(B, H, 128), _f64(bounds)
    kept = [paged.select(x[b], edges, pool.table[b], max(0, int(n)), page, select) for b, n in enumerate(pool.lens)]
    want_places = [[row + [-1] * (select - len(row)) for row in k] for k in kept]
    assert np.array_equal(places.cpu().numpy(), want_places), label
    K, V = pool.values()
    want = paged.decode_selected(x, K, V, pool.table, pool.lens, kept, **kw)
    got = bits(o).reshape(want.shape)
    live = pool.lens > 0
    assert not got[~live].any()
    if live.any():
        assert_parity(got[live], block.bf16_round_exact(want[live]), label, per_row_scales=True)
    assert torch.equal(call().view(torch.int16), o.view(torch.int16))


@pytest.mark.parametrize("kind", ["bf16", "e4m3", "block"])
@pytest.mark.parametrize("select", [1, 2, 7, 12, 13, 40])
def test_sparse_selections(kind, select):
    """Sequences with fewer pages than selected, as many, and more; empty ones and negative lengths among them."""
    announce("sparse", kind, select)
    rng = np.random.default_rng(select)
    _check_sparse(rng, kind, [200, 0, 1, 192, 193, 16 * 12, 16 * 12 + 1, 333, -4, 15], 10, 2, 16, select, label=f"{kind} {select}")


@pytest.mark.parametrize("H,n_kv", [(1, 1), (4, 2), (5, 1), (6, 1), (8, 1), (11, 1), (40, 8), (40, 2), (33, 1)])
def test_sparse_head_groups(H, n_kv):
    announce("sparse_heads", H, n_kv)
    _check_sparse(np.random.default_rng(H), "block", [500, 33, 700], H, n_kv, 32, 4, label=f"{H}/{n_kv}")


@pytest.mark.parametrize("kind,page,lens,select", [("bf16", 64, [9000, 130], 9), ("block", 16, [60] * 130 + [900], 5),
                                                   ("e4m3", 256, [20000], 3), ("block", 16, [150000], 60), ("bf16", 32, [40000, 70], 1100)])
def test_sparse_sizes(kind, page, lens, select):
    """Many sequences, many pages (more than are kept in LDS while they are chosen from), many selected."""
    announce("sparse_sizes", kind, page, len(lens), select)
    _check_sparse(np.random.default_rng(page), kind, lens, 4, 1, page, select, label=f"{kind} {page}", layout="heads")


def test_sparse_selects_as_many_as_the_type_counts():
    announce("sparse_most")
    n = 2 ** 31 - 1
    g = torch.Generator().manual_seed(74)
    k, v = (torch.randn(4, 1, 16, 128, generator=g).bfloat16().to(DEV) for _ in range(2))
    q = torch.randn(1, 128, generator=g).bfloat16().to(DEV)
    table, lens = torch.tensor([[2, 0, 3]], dtype=torch.int32, device=DEV), torch.tensor([40], dtype=torch.int32, device=DEV)
    bounds = torch.zeros(4, 1, 2, 128, dtype=torch.bfloat16, device=DEV)
    places = torch.empty(n + 1, dtype=torch.int32, device=DEV).fill_(7)        # (one behind the last)
    got = ops.sdpa_decode_paged_sparse(q, k, v, table, lens, bounds, n, selected=places[:n].view(1, 1, n))
    few = ops.sdpa_decode_paged_sparse(q, k, v, table, lens, bounds, 3)
    assert torch.equal(got, few)
    assert places[:4].tolist() == [0, 1, 2, -1] and int(places[-1]) == 7
    assert all(bool((part == -1).all()) for part in places[3:n].split(2 ** 28))


@pytest.mark.parametrize("layout", ["tokens", "slice"])
def test_sparse_layouts_and_scales(layout):
    announce("sparse_layout", layout)
    rng = np.random.default_rng(71)
    _check_sparse(rng, "block", [300, 90], 8, 2, 32, 3, layout=layout, scale=0.3)
    _check_sparse(rng, "bf16", [300, 90], 8, 2, 32, 3, layout=layout, qscale=0.0)       # all scores equal: the earliest pages


def test_sparse_ties_and_bounds_that_are_not_finite():
    """Equal bounds: the earlier page; NaN first, then infinities; -0 as 0."""
    announce("sparse_ties")
    rng = np.random.default_rng(72)

    def few(pool):                                        # every page one of three bounds
        kinds = _rand_bits(rng, 3, 1, 2, 128)
        return kinds[rng.integers(0, 3, pool.k.shape[0])].repeat(2, axis=1)

    _check_sparse(rng, "bf16", [900, 250], 8, 2, 16, 20, bounds=few)

    def zeros(pool):
        return rng.choice(np.array([0, 0x8000], np.uint16), (pool.k.shape[0], 2, 2, 128))

    _check_sparse(rng, "bf16", [900, 250], 8, 2, 16, 20, bounds=zeros)

    def odd(pool):
        x = np.sort(_f64(_rand_bits(rng, pool.k.shape[0], 2, 2, 128)), axis=2)
        x = block.bf16_round_exact(x)
        x[pool.table[0, 5], 0, :, 3] = NAN_BF16
        x[pool.table[0, 9], 1, 0, 64] = NAN_BF16
        x[pool.table[1, 3], 0, 1, 10] = 0x7F80
        return x

    _check_sparse(rng, "bf16", [900, 250], 2, 2, 16, 4, bounds=odd)


def test_sparse_counts_close_scores_exactly():
    """Pages whose scores differ in the last bits that bf16 bounds allow, and bounds far apart in magnitude."""
    announce("sparse_close")
    rng = np.random.default_rng(73)

    def close(pool):
        x = np.ones((pool.k.shape[0], 1, 2, 128))
        x[:, 0, 0] = -1
        x[np.arange(len(x)), 0, 1, rng.integers(0, 128, len(x))] += 2.0 ** -7
        x[:, 0, 1, 0] = 2.0 ** rng.integers(8, 10, len(x))
        return block.bf16_round_exact(x)

    _check_sparse(rng, "bf16", [3000], 3, 1, 16, 50, bounds=close, qscale=1.0)


@pytest.mark.parametrize("select", [2, 9, 600, 1249])
def test_sparse_counts_crowded_scores(select):
    """Many equal scores, more than are ranked one by one; scores crowded beside one far above, or NaN, or far below."""
    announce("sparse_crowded", select)
    rng = np.random.default_rng(select)

    def few(pool):
        return np.sort(_rand_bits(rng, 3, 1, 2, 128), axis=2)[rng.integers(0, 3, pool.k.shape[0])]

    def beside(value, page):
        def make(pool):
            x = rng.standard_normal((pool.k.shape[0], 1, 1, 128)) * 2.0 ** -6 + np.array([-1.0, 1.0]).reshape(2, 1)
            x = block.bf16_round_exact(x)
            x[pool.table[0, page], 0, :, 3] = value
            return x
        return make

    for bounds in (few, beside(NAN_BF16, 77), beside(0x7F00, 1000), beside(0xFF00, 3)):
        _check_sparse(rng, "bf16", [20000], 4, 1, 16, select, bounds=bounds, qscale=1.0)


def test_sparse_bad_pages_and_lengths_are_reported():
    """A page id out of range, scored or attended, a length past the table: NaN there and NMI_ERR_ASYNC once; the others
    right."""
    rng = np.random.default_rng(74)
    pool = BlockPool(rng, [300, 400, 90], 2, 16)
    bounds = _dev(block.bf16_round_exact(np.nan_to_num(paged.page_bounds(_f32_keys(pool)))))
    q = _dev(_rand_bits(rng, 3, 8 * 128, scale=0.3))

    def run(table, lens):
        return bits(ops.sdpa_decode_paged_sparse(q, pool.dk, pool.dv, _dev(table), _dev(lens), bounds, 4, k_scale=pool.dks,
                                                 v_scale=pool.dvs))

    good = run(pool.table, pool.lens)
    for change in ("page", "negative", "newest", "length"):
        announce("sparse_bad", change)
        table, lens = pool.table.copy(), pool.lens.copy()
        if change == "length":
            lens[1] = table.shape[1] * 16 + 1
        else:
            table[1, 24 if change == "newest" else 7] = -1 if change == "negative" else pool.k.shape[0]
        got = run(table, lens)
        torch.cuda.synchronize()
        assert np.isnan(_f64(got[1])).all()
        if change == "length":                             # (as above: the tiles are dealt otherwise)
            assert_parity(got[[0, 2]], good[[0, 2]], change)
        else:
            assert np.array_equal(got[[0, 2]], good[[0, 2]])
        assert _lib.lib().nmi_async_status() == _lib.NMI_ERR_ASYNC and _lib.lib().nmi_async_status() == 0
    assert np.array_equal(run(pool.table, pool.lens), good)


@pytest.mark.parametrize("select", [2, 30])
def test_sparse_strides_and_outputs(select):
    """q and o as columns of wider buffers; the rest of o's buffer stays as it was."""
    announce("sparse_strides", select)
    rng = np.random.default_rng(76)
    pool = BlockPool(rng, [1000, 5, 0], 2, 32)
    bounds = _dev(block.bf16_round_exact(np.nan_to_num(paged.page_bounds(_f32_keys(pool)))))
    wide = torch.full((3, 8 * 128 + 72), 9.0, dtype=torch.bfloat16, device=DEV)
    wide[:, 8:8 + 1024] = _dev(_rand_bits(rng, 3, 8 * 128))
    out = torch.full((3, 8 * 128 + 6), 7.0, dtype=torch.bfloat16, device=DEV)
    args = (pool.dk, pool.dv, pool.dtable, _dev(pool.lens), bounds, select)
    got = ops.sdpa_decode_paged_sparse(wide[:, 8:1032], *args, k_scale=pool.dks, v_scale=pool.dvs, out=out[:, 2:1026])
    alone = ops.sdpa_decode_paged_sparse(wide[:, 8:1032].contiguous(), *args, k_scale=pool.dks, v_scale=pool.dvs)
    assert _same(got, alone) and not alone[2].any() and alone[:2].any()
    assert (out[:, :2] == 7).all() and (out[:, 1026:] == 7).all()


def test_sparse_takes_its_workspace_from_the_allocator():
    import ctypes

    announce("sparse_bump")
    rng = np.random.default_rng(75)
    pool = BlockPool(rng, [900, 5], 4, 16)
    bounds = _dev(block.bf16_round_exact(np.nan_to_num(paged.page_bounds(_f32_keys(pool)))))
    q, lens = _dev(_rand_bits(rng, 2, 16 * 128)), _dev(pool.lens)
    want = ops.sdpa_decode_paged_sparse(q, pool.dk, pool.dv, pool.dtable, lens, bounds, 9, k_scale=pool.dks, v_scale=pool.dvs)
    c = _lib.PagedKv(pool.dk.data_ptr(), pool.dv.data_ptr(), 4 * 16 * 128, 16 * 128, 128, pool.dtable.data_ptr(),
                     pool.table.shape[1], pool.dks.data_ptr(), pool.dvs.data_ptr(), 2, pool.dk.shape[0], 16, pool.table.shape[1], 4)
    L, got = _lib.lib(), torch.zeros_like(want)
    rc = L.nmi_sdpa_decode_paged_sparse(ctypes.addressof(c), q.data_ptr(), 16 * 128, got.data_ptr(), 16 * 128, lens.data_ptr(),
                                        bounds.data_ptr(), 9, None, 2, 16, 128 ** -0.5, None, 0, torch.cuda.current_stream().cuda_stream)
    assert rc == 0, L.nmi_last_error()
    torch.cuda.synchronize()
    assert torch.equal(got.view(torch.int16), want.view(torch.int16)) and L.nmi_alloc_rewind() in (0, None)


# --- pages handed out ------------------------------------------------------------------------------


def _requests(rng, batch, width, page, n_pages, most, used=0.5):
    """Lengths that hold scattered pages, a table, a stack of the others, and new tokens of every kind."""
    lens = rng.integers(-1, int(width * page * used) + 1, batch)
    have = [-(-max(0, int(n)) // page) for n in lens]
    while sum(have) > n_pages:
        b = int(np.argmax(have))
        lens[b], have[b] = 0, 0
    ids = rng.permutation(n_pages).astype(np.int32)
    table = rng.integers(-5, n_pages + 5, (batch, width)).astype(np.int32)      # what is not in use: anything
    at = 0
    for b, n in enumerate(have):
        table[b, :n] = ids[at:at + n]
        at += n
    new = rng.integers(0, most + 1, batch)
    new[rng.random(batch) < 0.15] = -1
    new[rng.random(batch) < 0.1] = -2 ** 31
    free = np.full(n_pages, -9, np.int32)
    free[:n_pages - at] = ids[at:]
    return lens.astype(np.int32), new.astype(np.int32), table, free, n_pages - at


def _check_assign(lens, new, table, free, count, page, packed, extra_rows=0, wide=0):
    want_table, want_free = [list(r) for r in table], list(free)
    want = paged.assign(lens, new, want_table, want_free, count, page, packed)
    store = torch.full((len(lens), table.shape[1] + wide), -77, dtype=torch.int32, device=DEV)
    store[:, :table.shape[1]] = _dev(table)
    dtable, dfree = store[:, :table.shape[1]], _dev(free)
    tokens = want["cu_seqlens"][-1] + extra_rows if packed else None
    dlens, dcount = _dev(lens), _dev(np.array([count], np.int32))
    got = ops.kv_assign_paged(dlens, None if new is None else _dev(new), dtable, dfree, dcount, page, tokens=tokens)
    torch.cuda.synchronize()
    assert _lib.lib().nmi_async_status() == 0
    if packed:
        want["slots"] = want["slots"] + [-1] * extra_rows
    for name, value in got._asdict().items():
        if want[name] is None:
            assert value is None
        else:
            assert value.tolist() == want[name], name
    assert np.array_equal(dtable.cpu().numpy(), np.array(want_table)) and dfree.tolist() == [int(i) for i in want_free]
    assert (store[:, table.shape[1]:] == -77).all()
    assert dlens.tolist() == list(lens) and int(dcount) == count                # inputs stay
    return got


@pytest.mark.parametrize("batch", [1, 2, 63, 64, 65, 1000, 1023, 1024, 1025, 3000])
@pytest.mark.parametrize("page", [16, 128])
def test_assign(batch, page):
    announce("assign", batch, page)
    rng = np.random.default_rng(batch + page)
    for n_pages, most in ((4 * batch + 3, 1), (4 * batch + 3, 3 * page), (batch // 2 + 1, page + 1), (8 * batch, 5)):
        r = _requests(rng, batch, 6, page, n_pages, most)
        _check_assign(*r, page, True, extra_rows=int(rng.integers(0, 70)), wide=3)
        lens, new, *rest = _requests(rng, batch, 6, page, n_pages, 1)
        _check_assign(lens, new, *rest, page, False)
        _check_assign(lens, None, *rest, page, False, wide=1)


def test_assign_edges():
    """Nothing free, everything asked for, rows of one page, sequences at the end of their rows, one long prompt."""
    rng = np.random.default_rng(81)
    announce("assign_edges")
    table = lambda b, w: rng.integers(0, 9, (b, w)).astype(np.int32)  # noqa: E731
    i32 = lambda *x: np.array(x, np.int32)  # noqa: E731
    free = np.arange(9, dtype=np.int32)
    _check_assign(i32(16, 15, 0, -1), i32(1, 1, 1, 1), table(4, 2), free, 0, 16, False)
    _check_assign(i32(0, 0, 0), i32(16 * 4, 16 * 5, 1), table(3, 9), free, 9, 16, True)
    _check_assign(i32(0, 0, 3), i32(16 * 10, 1, 14), table(3, 9), free, 9, 16, True)         # too long for its row: asks for nothing
    _check_assign(i32(16, 15), i32(1, 1), table(2, 1), free, 9, 16, False)
    _check_assign(i32(0), i32(60000), np.zeros((1, 470), np.int32), rng.permutation(480).astype(np.int32), 480, 128, True)
    _check_assign(i32(0, 5), i32(0, 0), table(2, 3), free, 9, 16, True, extra_rows=0)        # no rows at all
    _check_assign(i32(40, 5), i32(-1, -1), table(2, 3), free, 3, 16, True, extra_rows=2)
    _check_assign(i32(2 ** 30 - 1), i32(1), table(1, 1024), free, 9, 1 << 20, False)
    _check_assign(i32(2 ** 30 - 1), i32(2), table(1, 1024), free, 9, 1 << 20, True)


@pytest.mark.parametrize("change", ["count_high", "count_low", "long", "long_ended", "two_rows", "cut", "bad_page", "bad_push", "overflow", "huge"])
def test_assign_bad_data_is_cut_and_reported(change):
    """What is out of range is never followed: buffers stay within their guards, the other sequences get what the rule
    gives them, and NMI_ERR_ASYNC says so once."""
    announce("assign_bad", change)
    page, n_pages, batch, width = 16, 12, 4, 3
    lens, new = np.array([20, 16, 0, 40], np.int32), np.array([1, 1, 1, 1], np.int32)
    table = np.array([[0, 1, -1], [2, -1, -1], [-1, -1, -1], [3, 4, 5]], np.int32)
    free, count, packed, tokens = np.array([6, 7, 8, 9, 10, 11] + [-1] * 6, np.int32), 6, False, None
    good = [0, 1, 2, 3]
    if change == "count_high":
        free[6:] = [0] * 6
        count, good = 100, [0, 3]
    elif change == "count_low":
        count, good = -5, [0, 3]
    elif change == "long":
        lens[3], good = 49, [0, 1, 2]
    elif change == "long_ended":
        lens[3], new[3], good = 2 ** 31 - 1, -1, [0]
    elif change == "two_rows":
        new[3], good = 2, [0, 1, 2]
    elif change == "cut":
        packed, tokens, good = True, 3, [0, 1, 2]
    elif change == "bad_page":
        table[0, 1], good = 12, [1, 2, 3]
    elif change == "bad_push":
        new[3], table[3, 1], good = -1, -3, [0]
    elif change == "overflow":
        free[6:], count = 0, 11
        new[3], good = -1, [0]
    else:
        packed, tokens, good = True, 4, [0]
        new[1:] = 2 ** 31 - 1
    guard = 5
    flat = torch.full((batch * width + 2 * guard,), -77, dtype=torch.int32, device=DEV)
    flat[guard:-guard] = _dev(table).flatten()
    dtable = flat[guard:-guard].view(batch, width)
    stack = torch.full((n_pages + 2 * guard,), -77, dtype=torch.int32, device=DEV)
    stack[guard:-guard] = _dev(free)
    got = ops.kv_assign_paged(_dev(lens), _dev(new), dtable, stack[guard:-guard], _dev(np.array([count], np.int32)), page, tokens=tokens)
    torch.cuda.synchronize()
    assert _lib.lib().nmi_async_status() == _lib.NMI_ERR_ASYNC and _lib.lib().nmi_async_status() == 0
    for t in (flat, stack):
        assert (t[:guard] == -77).all() and (t[-guard:] == -77).all()
    want = paged.assign([int(n) for n in np.where(np.isin(range(4), good), lens, -1)], np.minimum(new, 99), [list(r) for r in table], list(free),
                        min(max(count, 0), n_pages), page, packed)
    for b in good:
        assert int(got.lens[b]) == want["lens"][b] and int(got.kv_lens[b]) == want["kv_lens"][b]
        if change not in ("long_ended", "bad_push", "overflow", "count_high"):
            assert int(got.slots[b]) == want["slots"][b]
    assert 0 <= int(got.free_count) <= n_pages
    assert got.slots.min() >= -1 and got.slots.max() < n_pages * page
    if packed:
        assert (got.cu_seqlens.diff() >= 0).all() and int(got.cu_seqlens[-1]) <= tokens


# --- together --------------------------------------------------------------------------------------


class Server:
    """Conversations on one pool: pages assigned, prompts and tokens appended, pages bounded, selected, attended."""

    def __init__(self, kind, batch=6, n_pages=40, width=12, page=32, H=8, n_kv=2, select=3):
        self.kind, self.batch, self.page, self.H, self.n_kv, self.select = kind, batch, page, H, n_kv, select
        type_ = torch.bfloat16 if kind == "bf16" else torch.float8_e4m3fn
        self.k, self.v = (torch.zeros(n_pages, n_kv, page, 128, device=DEV).to(type_) for _ in range(2))
        shape = {"bf16": None, "e4m3": (n_kv,), "block": (n_pages, n_kv, page // 16)}[kind]
        self.ks, self.vs = (None if shape is None else torch.full(shape, 0.01, device=DEV) for _ in range(2))
        self.bounds = torch.zeros(n_pages, n_kv, 2, 128, dtype=torch.bfloat16, device=DEV)
        self.table = torch.full((batch, width), -1, dtype=torch.int32, device=DEV)
        self.free, self.count = torch.arange(n_pages, dtype=torch.int32, device=DEV), torch.tensor([n_pages], dtype=torch.int32, device=DEV)
        self.lens = torch.zeros(batch, dtype=torch.int32, device=DEV)
        self.freq = 10000.0 ** (-torch.arange(0, 64, 2, device=DEV, dtype=torch.float32) / 64)
        self.new = torch.zeros(batch, dtype=torch.int32, device=DEV)
        self.out, self.all = (torch.zeros(batch, H * 128, dtype=torch.bfloat16, device=DEV) for _ in range(2))
        self.x = torch.zeros(batch, (H + 2 * n_kv) * 128, dtype=torch.bfloat16, device=DEV)

    def step(self, x, tokens=None):
        q, k, v = x.split([self.H * 128, self.n_kv * 128, self.n_kv * 128], dim=1)
        scales = dict(k_scale=self.ks, v_scale=self.vs)
        s = ops.kv_assign_paged(self.lens, self.new, self.table, self.free, self.count, self.page, tokens=tokens,
                                lens_out=self.lens, free_count_out=self.count)
        q, _ = ops.kv_append_paged(k, v, self.k, self.v, self.table, s.start_pos, cu_seqlens=s.cu_seqlens, q=q, inv_freq=self.freq, **scales)
        ops.kv_bounds_paged(self.k, self.table, s.start_pos, self.bounds, cu_seqlens=s.cu_seqlens, tokens=tokens, k_scale=self.ks)
        if tokens is None:
            ops.sdpa_decode_paged(q, self.k, self.v, self.table, s.kv_lens, out=self.all, **scales)
            ops.sdpa_decode_paged_sparse(q, self.k, self.v, self.table, s.kv_lens, self.bounds, self.select, out=self.out, **scales)
        return s, q

    def state(self):
        return [t for t in (self.k, self.v, self.ks, self.vs, self.bounds, self.table, self.free, self.count, self.lens, self.out, self.all)
                if t is not None]


def _same(a, b):
    return a.dtype == b.dtype and torch.equal(a.contiguous().view(torch.uint8), b.contiguous().view(torch.uint8))


@pytest.mark.parametrize("kind", ["bf16", "e4m3", "block"])
def test_prompts_then_steps(kind):
    """Prompts, then steps of one token in which conversations end and others start: every output against the oracle fed
    with the true cache, its owners' pages apart."""
    announce("step", kind)
    rng = np.random.default_rng(90)
    s = Server(kind)
    lens = [200, 3, 64, 31, 130, 90]
    s.new.copy_(_dev(np.array(lens, np.int32)))
    s.step(_dev(_rand_bits(rng, sum(lens), 12 * 128)), tokens=sum(lens))
    for step in range(40):
        new = np.ones(6, np.int32)
        if step % 9 == 4:
            new[step % 6] = -1                             # one ends
        if step % 5 == 2:
            new[(step + 1) % 6] = 0                        # one waits
        s.new.copy_(_dev(new))
        got, q = s.step(_dev(_rand_bits(rng, 6, 12 * 128)))
        torch.cuda.synchronize()
        held = got.lens.cpu().numpy()
        table = s.table.cpu().numpy()
        own = [table[b, i] for b in range(6) for i in range(-(-max(0, held[b]) // 32))]
        assert sorted(own + s.free[:int(s.count)].tolist()) == list(range(40))
        kv = got.kv_lens.cpu().numpy()
        if kind == "bf16":
            K, V = _f64(bits(s.k)), _f64(bits(s.v))
        else:
            spread = (lambda t: t.cpu().numpy()[None, :, None, None]) if kind == "e4m3" else \
                (lambda t: np.repeat(t.cpu().numpy(), 16, axis=2)[..., None])
            K, V = (np.nan_to_num(LUT[c.view(torch.uint8).cpu().numpy()] * spread(x)) for c, x in ((s.k, s.ks), (s.v, s.vs)))
        x = _f64(bits(q)).reshape(6, 8, 128)
        live = kv > 0
        want = paged.decode(x, K, V, table, kv)
        assert_parity(bits(s.all).reshape(want.shape)[live], block.bf16_round_exact(want[live]), f"{kind} {step}")
        edges = _f64(bits(s.bounds))
        for b in np.flatnonzero(live):                     # complete pages have the bounds of what they hold
            ids = table[b, :kv[b] // 32]
            assert np.array_equal(edges[ids], _bf16(paged.page_bounds(K[ids].astype(np.float32).astype(np.float64))))
        kept = [paged.select(x[b], edges, table[b], int(kv[b]), 32, 3) for b in range(6)]
        want = paged.decode_selected(x, K, V, table, kv, kept)
        assert_parity(bits(s.out).reshape(want.shape)[live], block.bf16_round_exact(want[live]), f"{kind} {step} selected")
        assert not s.out[~torch.from_numpy(live).to(DEV)].any()
        ended = np.flatnonzero(held < 0)
        if len(ended):                                     # another conversation starts in its place
            s.lens[int(ended[0])] = 0
    assert _lib.lib().nmi_async_status() == 0


@pytest.mark.parametrize("n_pages", [25, 19])
@pytest.mark.parametrize("kind", ["bf16", "block"])
def test_a_captured_step_goes_on_as_sequences_grow_and_end(kind, n_pages):
    """One graph of the whole step, replayed with eager steps on a second server between the replays: everything that
    they hold is equal, byte for byte, over page borders, ends and new starts, with pages enough and too few."""
    announce("step_graph", kind, n_pages)
    rng = np.random.default_rng(91)
    a, b = Server(kind, n_pages=n_pages), Server(kind, n_pages=n_pages)
    lens = [100, 3, 64, 31, 130, 90]
    x = _dev(_rand_bits(rng, sum(lens), 12 * 128))
    for s in (a, b):
        s.new.copy_(_dev(np.array(lens, np.int32)))
        s.step(x, tokens=sum(lens))
        s.new.fill_(0)
        s.step(s.x)                                        # (a step of no tokens, before the capture)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=torch.cuda.Stream()):
        a.step(a.x)
    granted = 0
    for i in range(150):
        new = np.ones(6, np.int32)
        if i % 20 == 19:
            new[i // 20 % 6] = -1
        x = _dev(_rand_bits(rng, 6, 12 * 128, scale=2.0 ** (i % 5 - 2)))
        for s in (a, b):
            s.new.copy_(_dev(new))
            s.x.copy_(x)
            s.out.fill_(9.0), s.all.fill_(9.0)
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        got, _ = b.step(b.x)
        torch.cuda.synchronize()
        assert all(_same(p, q) for p, q in zip(a.state(), b.state())), i
        granted += int((got.kv_lens > 0).sum())
        for s in (a, b):
            s.lens[s.lens < 0] = 0
    assert (granted == 150 * 6 - 7) == (n_pages == 25) and granted > 400       # (7 end)
    assert _lib.lib().nmi_async_status() == 0


def test_two_streams_and_two_threads():
    announce("step_streams")
    servers = [Server("block") for _ in range(4)]
    xs = [_dev(_rand_bits(np.random.default_rng(92), 6, 12 * 128)) for _ in range(30)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(4)]

    def work(i):
        with torch.cuda.stream(streams[i]):
            servers[i].new.fill_(1)
            for _ in range(3):
                for x in xs:
                    servers[i].step(x)

    work(0)
    torch.cuda.synchronize()
    work(1)                                                # streams in turn from one thread: no waits between them
    threads = [threading.Thread(target=work, args=(i,)) for i in (2, 3)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    for s in servers[1:]:
        assert all(_same(p, q) for p, q in zip(s.state(), servers[0].state()))
    assert int(servers[0].lens[0]) == 90


def test_assign_grants_nothing_to_a_step_of_no_rows():
    """Sequences end; one that asks for a token all the same is out of range."""
    announce("assign_no_rows")

    def ints(*v):
        return torch.tensor(v, dtype=torch.int32, device=DEV)

    table, free, count = torch.tensor([[0, 1], [2, 9], [3, 9]], dtype=torch.int32, device=DEV), ints(4, 5, 6, 7, 8, 8, 8, 8), ints(2)
    got = ops.kv_assign_paged(ints(20, 16, 3), ints(-1, 0, 0), table, free, count, 16, tokens=0)
    assert [t.tolist() for t in got] == [[-1] * 3, [0] * 3, [0] * 4, [], [-1, 16, 3], [4]]
    assert free.tolist() == [4, 5, 0, 1, 8, 8, 8, 8]
    torch.cuda.synchronize()
    got = ops.kv_assign_paged(ints(-1, 16, 3), ints(0, 1, 0), table, free, ints(4), 16, tokens=0)
    assert [t.tolist() for t in got] == [[-1] * 3, [0] * 3, [0] * 4, [], [-1, 16, 3], [4]]
    assert table.tolist() == [[0, 1], [2, 9], [3, 9]]
    torch.cuda.synchronize()
    with pytest.raises(_lib.NmiError):
        ops.kv_assign_paged(ints(-1), ints(0), table[:1], free, ints(4), 16, tokens=0)


def test_the_front_end_keeps_nothing():
    announce("step_front")
    s = Server("block")
    x = _dev(_rand_bits(np.random.default_rng(93), 6, 12 * 128))
    s.new.fill_(0)
    places = torch.zeros(6, 2, 3, dtype=torch.int32, device=DEV)

    def once():
        got, q = s.step(x)
        refs = sys.getrefcount(q), sys.getrefcount(got.start_pos), sys.getrefcount(got.slots)      # (an assert holds its operands)
        assert refs == (2, 2, 2) and got.cu_seqlens is None
        assert got.lens is s.lens and got.free_count is s.count
        ops.kv_assign_paged(s.lens, s.new, s.table, s.free, s.count, 32, tokens=0)
        ops.sdpa_decode_paged_sparse(q, s.k, s.v, s.table, s.lens, s.bounds, 3, k_scale=s.ks, v_scale=s.vs, selected=places)

    once()
    torch.cuda.synchronize()
    held = [*s.state(), s.new, s.freq, x, places]
    counts, memory, nones = [sys.getrefcount(t) for t in held], torch.cuda.memory_allocated(), sys.getrefcount(None)
    for _ in range(200):
        once()
    torch.cuda.synchronize()
    assert [sys.getrefcount(t) for t in held] == counts and torch.cuda.memory_allocated() == memory
    assert abs(sys.getrefcount(None) - nones) < 100
    for _ in range(3):
        with pytest.raises(_lib.NmiError, match="page_size=8"):
            ops.kv_assign_paged(s.lens, s.new, s.table, s.free, s.count, 8)
        with pytest.raises(ValueError, match="no pages"):
            ops.kv_assign_paged(s.lens, s.new, s.table[:, :0], s.free, s.count, 16)
    assert [sys.getrefcount(t) for t in held] == counts


def test_e4m3_codes_of_the_oracle():
    """(e4m3's table has each value once but for the zeros, so that values compare codes.)"""
    lut = e4m3.decode_lut()
    assert len(np.unique(lut[np.isfinite(lut)])) == 253
