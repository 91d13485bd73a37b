"""GPU tests of batched attention serving where its device data is out of order or range, and where values
are not finite.  Bars as in test_paged_gpu.py: what is copied is bit for bit, attention goes by the parity
gate of oracle.linear.parity against float64 rounded once."""
import numpy as np
import pytest
import torch

from nemotron_infer_amd import _lib, ops
from oracle import block, paged
from tests.gpu_util import announce, assert_parity, bits
from tests.test_paged_gpu import LUT, NAN_BF16, Pool, _bf16, _between, _dev, _f64, _rand_bits

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _no_pending_error():
    _lib.lib().nmi_async_status()
    yield
    torch.cuda.synchronize()
    _lib.lib().nmi_async_status()


def _cut(cu, T):
    """[(first, end)] of the sequences, cut to the T rows; (0, 0) for offsets that fall."""
    return [(min(max(int(a), 0), T), max(min(max(int(a), 0), T), min(max(int(b), 0), T))) for a, b in zip(cu, cu[1:])]


BAD_OFFSETS = [
    (50, [0, 20, 51]), (50, [-1, 20, 50]), (50, [0, 30, 20]), (50, [0, 20, 10, 50]), (12, [0, 8, 2, 4, 12]),
    (50, [2 ** 31 - 1] * 3), (50, [-5, -5, -5]), (50, [-2 ** 31, 50]), (50, [60, 70]),
    (50, [3, 20, 40, 2 ** 31 - 1, 40]),
    # more sequences than lanes: behind the rows' own, before them, and between
    (10, [0, 5, 10] + [10] * 100 + [11]), (10, [0, 5, 10] + [10] * 100 + [9]), (10, [0, -1] + [0] * 100 + [4, 10]),
    (300, [*range(0, 150), 100, *range(150, 301)]),
]


@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
@pytest.mark.parametrize("rotary", [0, 128])
@pytest.mark.parametrize("T,cu", BAD_OFFSETS, ids=[str(i) for i in range(len(BAD_OFFSETS))])
def test_append_bad_offsets_are_cut_and_reported(kind, rotary, T, cu):
    """Offsets that fall or leave the rows are cut to them, as for the attention over packed prompts: the rows of
    each sequence from its first on, a row that several have as the first one's; rows of none are not
    stored or returned, and NMI_ERR_ASYNC says so once."""
    announce("append_bad_offsets", kind, rotary, T, cu[:8])
    rng = np.random.default_rng(T + len(cu))
    n_kv, H, page, batch = 2, 4, 16, len(cu) - 1
    starts = rng.integers(0, 40, batch).astype(np.int32)
    spans = _cut(cu, T)
    pool = Pool(rng, [int(s) for s in starts], n_kv, page, kind,
                hold=[int(s) + b - a for s, (a, b) in zip(starts, spans)])
    q, k, v = (_rand_bits(rng, T, n * 128) for n in (H, n_kv, n_kv))
    before = [pool.host(pool.dk).copy(), pool.host(pool.dv).copy()]
    f = (10000.0 ** (-np.arange(64) / 64)).astype(np.float32) if rotary else None
    qo = torch.full((T, H * 128), 5.0, dtype=torch.bfloat16, device="cuda") if rotary else None
    ko = torch.full((T, n_kv * 128), 5.0, dtype=torch.bfloat16, device="cuda") if rotary else None
    ops.kv_append_paged(_dev(k), _dev(v), pool.dk, pool.dv, pool.dtable, _dev(starts), cu_seqlens=_dev(np.array(cu)),
                        q=_dev(q) if rotary else None, inv_freq=_dev(f) if rotary else None, k_scale=pool.dks,
                        v_scale=pool.dvs, q_out=qo, k_out=ko)
    torch.cuda.synchronize()
    assert _lib.lib().nmi_async_status() == _lib.NMI_ERR_ASYNC
    assert _lib.lib().nmi_async_status() == 0
    rows = [(t, b, int(starts[b]) + t - spans[b][0]) for t in range(T)
            for b in [next((i for i, (x, y) in enumerate(spans) if x <= t < y), -1)] if b >= 0]
    after = [pool.host(pool.dk), pool.host(pool.dv)]
    stored = np.zeros(before[0].shape, bool)
    if rows:
        r, seq, pos = (np.array(x) for x in zip(*rows))
        at = (pool.table[seq, pos // page], slice(None), pos % page)
        stored[at] = True
        vals = [_f64(x[r]).reshape(len(r), n_kv, 128) for x in (k, v)]
        slack = [0 * x for x in vals]
        if rotary:
            slack[0] = paged.partner_sum(vals[0], rotary, False) * 2.0 ** -20
            vals[0] = paged.rotate(vals[0], pos.astype(np.float64), f, False)
            x = _f64(q[r]).reshape(len(r), H, 128)
            _between(_f64(bits(qo)[r]).reshape(x.shape), paged.rotate(x, pos.astype(np.float64), f, False),
                     paged.partner_sum(x, rotary, False) * 2.0 ** -20, _bf16)
            _between(_f64(bits(ko)[r]).reshape(vals[0].shape), vals[0], slack[0], _bf16)
        for new, want, d, s in zip(after, vals, slack, (pool.ks, pool.vs)):
            if kind == "bf16":
                _between(_f64(new[at]), want, d, _bf16)
            else:
                sc = s.astype(np.float64)[:, None]
                _between(LUT[new[at]], want / sc, d / sc + np.abs(want / sc) * 2.0 ** -22, paged.round_e4m3)
    for new, old in zip(after, before):
        assert np.array_equal(new[~stored], old[~stored])
    if rotary:
        rest = np.setdiff1d(np.arange(T), [t for t, _, _ in rows])
        assert (qo.cpu()[rest] == 5).all() and (ko.cpu()[rest] == 5).all()


INF, NINF = 0x7F80, 0xFF80


@pytest.mark.parametrize("lens,H,n_kv,page", [([777], 40, 8, 16), ([1], 8, 2, 16), ([20, 33, 5], 6, 2, 16), ([20000, 33], 10, 2, 128),
                                              ([5] * 70 + [900] + [17] * 9, 8, 2, 32), ([40] * 300, 17, 1, 16),
                                              ([130] * 8, 8, 8, 64)],
                         ids=["777", "1", "3 short", "20000", "80", "300", "8"])
def test_decode_of_values_that_are_not_finite(lens, H, n_kv, page):
    """Infinities and NaN in single dims of v, in the first, the last and other positions that are attended: those
    dims' outputs are that infinity (of both signs: NaN) or NaN, as in the formula, since every weight is
    positive; all others as without."""
    announce("decode_not_finite", len(lens), max(lens), H, n_kv)
    rng = np.random.default_rng(sum(lens))
    pool = Pool(rng, lens, n_kv, page, "bf16")

    def put(b, pos, head, dims, value):
        pool.v[pool.table[b, pos // page], head, pos % page, dims] = value

    for b, n in enumerate(lens):
        if b % 3 == 1:
            continue                                       # (sequences without)
        put(b, n - 1, 0, [0, 127], INF)                     # whose row is read again for the rows past the end
        put(b, 0, n_kv - 1, [1, 64], NINF)
        put(b, n // 2, 0, [5, 6, 77], NINF)
        put(b, n // 3, 0, [77], INF)                        # with the one before: NaN (but for one position)
        put(b, int(rng.integers(0, n)), 0, [90], NAN_BF16)
        put(b, int(rng.integers(0, n)), n_kv - 1, [33, 34], 0x7F7F)     # the largest finite value: stays as it is
    pool.dv = pool._to_dev(pool.v)
    q = _rand_bits(rng, len(lens), H * 128, scale=0.5)
    o = pool.decode(_dev(q))
    torch.cuda.synchronize()
    K, V = pool.values()
    with np.errstate(all="ignore"):
        want = paged.decode(_f64(q).reshape(len(lens), H, 128), K, V, pool.table, pool.lens)
        rounded = block.bf16_round_exact(np.where(np.isfinite(want), want, 0))
    got = bits(o).reshape(want.shape)
    assert np.array_equal(np.isnan(_f64(got)), np.isnan(want))
    assert np.array_equal(np.isposinf(_f64(got)), np.isposinf(want)) and np.array_equal(np.isneginf(_f64(got)), np.isneginf(want))
    assert (np.isinf(want).sum() > 0) and np.isfinite(want).mean() > 0.8
    clean = np.isfinite(want)
    assert_parity(got[clean], rounded[clean], "the others")
    assert _lib.lib().nmi_async_status() == 0


@pytest.mark.parametrize("scale", [0.09, 0.5, 1.0, 2.5])
@pytest.mark.parametrize("lens", [[777], [64, 300, 33], [2000, 5]], ids=["777", "3", "2000"])
def test_decode_of_scores_of_minus_infinity(lens, scale):
    """Positions whose score is minus infinity have no weight, also where a tile, or all that a wave has of a
    sequence, holds no other, whatever the scale."""
    announce("decode_minus_infinity", lens, scale)
    rng = np.random.default_rng(60)
    H, n_kv, page = 8, 2, 16
    pool = Pool(rng, lens, n_kv, page, "bf16")
    for b, n in enumerate(lens):
        for pos in {*range(0, min(40, n - 1)), *range(96, min(260, n - 1)), *range(600, max(600, n - 1))}:
            pool.k[pool.table[b, pos // page], :, pos % page] = 0
            pool.k[pool.table[b, pos // page], :, pos % page, 0] = NINF
    pool.dk = pool._to_dev(pool.k)
    q = _rand_bits(rng, len(lens), H * 128, scale=0.3)
    q.reshape(len(lens), H, 128)[:, :, 0] = block.bf16_round_exact(np.array([0.5]))[0]
    o = pool.decode(_dev(q), scale=scale)
    torch.cuda.synchronize()
    K, V = pool.values()
    with np.errstate(all="ignore"):
        want = paged.decode(_f64(q).reshape(len(lens), H, 128), K, V, pool.table, pool.lens, scale=scale)
    assert np.isfinite(want).all()
    assert_parity(bits(o).reshape(want.shape), block.bf16_round_exact(want), f"scale {scale}")


def test_one_kv_head_in_either_order_of_heads_and_positions():
    """K and V whose strides differ only in the dimension of one KV head, a page table of one column with a
    column stride of its own: the bytes of the plain layout."""
    announce("one_kv_head")
    rng = np.random.default_rng(61)
    pool = Pool(rng, [40, 64, 7], 1, 64, "bf16")
    q = _dev(_rand_bits(rng, 3, 6 * 128))
    lens = _dev(pool.lens)
    want = pool.decode(q)
    other = pool.dv.transpose(1, 2).contiguous().transpose(1, 2)
    other = other.as_strided(other.shape, (64 * 128, 128, 128, 1))
    assert other.stride() != pool.dk.stride()
    table = pool.dtable[:, 0].contiguous().as_strided((3, 1), (1, 3))
    assert torch.equal(ops.sdpa_decode_paged(q, pool.dk, other, table, lens).view(torch.int16), want.view(torch.int16))
    k, v = (_dev(_rand_bits(rng, 3, 128)) for _ in range(2))
    at = _dev(np.array([40, 5, 7], np.int32))
    ops.kv_append_paged(k, v, pool.dk, other, table, at)
    ids = pool.dtable[:, 0].long()
    assert torch.equal(pool.dk[ids, 0, at.long()], k) and torch.equal(other[ids, 0, at.long()], v)


@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
@pytest.mark.parametrize("batch", [65, 200, 700])
def test_decode_bad_pages_and_lengths_of_many_sequences(kind, batch):
    """More sequences than lanes: pages outside the pool and lengths past the table give NaN in their own
    sequences, wherever those are, the others the same bytes, and one report."""
    announce("decode_many_bad", kind, batch)
    rng = np.random.default_rng(batch)
    lens = rng.integers(1, 90, batch)
    lens[[0, batch // 2, batch - 1]] = 150, 400, 95
    width = 30
    pool = Pool(rng, lens, 2, 16, kind, width=width)
    q = _dev(_rand_bits(rng, batch, 8 * 128))
    good = bits(pool.decode(q))
    assert _lib.lib().nmi_async_status() == 0
    for pages, longs in (([0], []), ([batch - 1], []), ([], [batch - 1]), ([3, 64, batch // 2], [1, batch - 2])):
        table, now = pool.table.copy(), pool.lens.copy()
        for i, b in enumerate(pages):
            table[b, (lens[b] - 1) // 16] = pool.k.shape[0] + i if i % 2 == 0 else -5
        for b in longs:
            now[b] = width * 16 + 1 if b % 2 else 2 ** 31 - 1
            table[b] = table[b, 0]                          # (the whole of its row is read)
        keep, pool.dtable = pool.dtable, _dev(table)
        got = bits(pool.decode(q, lens=now))
        pool.dtable = keep
        torch.cuda.synchronize()
        assert _lib.lib().nmi_async_status() == _lib.NMI_ERR_ASYNC and _lib.lib().nmi_async_status() == 0
        bad = np.zeros(batch, bool)
        bad[pages + longs] = True
        assert np.isnan(_f64(got[bad])).all()
        if longs:                                          # (a longer row deals the tiles out anew)
            assert_parity(got[~bad], good[~bad], f"{pages} {longs}")
        else:
            assert np.array_equal(got[~bad], good[~bad])
    assert np.array_equal(bits(pool.decode(q)), good)


@pytest.mark.parametrize("T,cu", [(T, cu) for T, cu in BAD_OFFSETS], ids=[str(i) for i in range(len(BAD_OFFSETS))])
def test_prefill_bad_offsets_leave_right_rows(T, cu):
    """What is left of offsets cut to the rows is attended as prompts of that length; the rows of no sequence
    stay as they were.  A row that falling offsets give to several sequences is one of theirs: not compared."""
    announce("packed_bad_rows", T, cu[:8])
    rng = np.random.default_rng(T + len(cu))
    H, n_kv = 4, 2
    q, k, v = (_rand_bits(rng, T, n * 128) for n in (H, n_kv, n_kv))
    out = torch.full((T, H * 128), 3.0, dtype=torch.bfloat16, device="cuda")
    ops.sdpa_prefill_packed_bf16(_dev(q), _dev(k), _dev(v), _dev(np.array(cu)), H, n_kv, out=out)
    torch.cuda.synchronize()
    assert _lib.lib().nmi_async_status() == _lib.NMI_ERR_ASYNC and _lib.lib().nmi_async_status() == 0
    spans = _cut(cu, T)
    of = np.array([sum(a <= t < b for a, b in spans) for t in range(T)])
    got = bits(out).reshape(T, H, 128)
    assert (out.cpu()[of == 0] == 3).all()
    for a, b in spans:
        if b > a:
            want = paged.prefill(*(_f64(x[a:b]).reshape(b - a, -1, 128) for x in (q, k, v)), [0, b - a])
            mine = of[a:b] == 1
            if mine.any():
                assert_parity(got[a:b][mine], block.bf16_round_exact(want[mine]), f"{cu[:8]} {a}:{b}")


@pytest.mark.parametrize("lens", [[200, 40, 33, 300], [1], [129, 1000], [31] * 40], ids=["4", "1", "1000", "40"])
def test_prefill_of_values_that_are_not_finite(lens):
    """Infinities and NaN in single dims of v: the outputs of those dims are that infinity (of both signs: NaN) or
    NaN from the value's row on, as in the formula, all others as without; early and late in a prompt, in
    the first and the last rows of a wave's 32."""
    announce("packed_not_finite_values", lens[:4])
    rng = np.random.default_rng(sum(lens))
    H, n_kv = 10, 2
    T, cu = sum(lens), np.concatenate([[0], np.cumsum(lens)]).astype(np.int32)
    q, k, v = (_rand_bits(rng, T, n * 128, scale=0.5 if n == H else 1.0) for n in (H, n_kv, n_kv))
    for a, n in zip(cu, lens):
        for at, dims, value in ((0, [0], INF), (n // 3, [127, 3], NINF), (n // 2, [3], INF), (min(31, n - 1), [8, 9], INF),
                                (min(64, n - 1), [40], NAN_BF16), (n - 1, [128 + 5], NINF), (n // 4 // 32 * 32, [128 + 6], INF)):
            v[a + at, dims] = value
    o = ops.sdpa_prefill_packed_bf16(_dev(q), _dev(k), _dev(v), _dev(cu), H, n_kv)
    torch.cuda.synchronize()
    with np.errstate(all="ignore"):
        want = paged.prefill(*(_f64(x).reshape(T, -1, 128) for x in (q, k, v)), cu)
        rounded = block.bf16_round_exact(np.where(np.isfinite(want), want, 0))
    got = bits(o).reshape(want.shape)
    assert np.array_equal(np.isnan(_f64(got)), np.isnan(want))
    assert np.array_equal(np.isposinf(_f64(got)), np.isposinf(want)) and np.array_equal(np.isneginf(_f64(got)), np.isneginf(want))
    clean = np.isfinite(want)
    assert_parity(got[clean], rounded[clean], "the others")


@pytest.mark.parametrize("scale", [0.09, 1.0, 2.5])
def test_prefill_of_scores_of_minus_infinity(scale):
    """Keys whose score is minus infinity have no weight, also where all of a block's are; rows that see no
    other key are NaN, as in the formula."""
    announce("packed_minus_infinity", scale)
    rng = np.random.default_rng(62)
    H, n_kv, lens = 4, 2, [300, 70, 40]
    T, cu = sum(lens), np.concatenate([[0], np.cumsum(lens)]).astype(np.int32)
    q, k, v = (_rand_bits(rng, T, n * 128, scale=0.3 if n == H else 1.0) for n in (H, n_kv, n_kv))
    q.reshape(T, H, 128)[:, :, 0] = block.bf16_round_exact(np.array([0.5]))[0]
    for t in (*range(0, 40), *range(64, 200), 305, 380, 381, 409):
        k[t] = 0
        k[t, [0, 128]] = NINF
    o = ops.sdpa_prefill_packed_bf16(_dev(q), _dev(k), _dev(v), _dev(cu), H, n_kv, scale=scale)
    torch.cuda.synchronize()
    with np.errstate(all="ignore"):
        want = paged.prefill(*(_f64(x).reshape(T, -1, 128) for x in (q, k, v)), cu, scale=scale)
    got = bits(o).reshape(want.shape)
    assert np.isnan(want[:40]).all() and np.isfinite(want[40:]).all()
    assert np.isnan(_f64(got[:40])).all()
    assert_parity(got[40:], block.bf16_round_exact(want[40:]), f"scale {scale}")
