"""GPU tests of a serving step on a paged cache where it is easiest to get wrong: page scores that only one side of a
bound enters, a choice of one page, more pages coming back than there are.

Bars (derived before the first run): selected places are whole numbers, equal to those of the oracle, whose scores are
sums in 64 bits rounded to float32 once as the kernel's are; in another order, so that two scores may change places only if
they lie within 128 * 2^-53 of the sum of their terms' magnitudes of one another, which random ordinary terms do not.
"""
import ctypes

import numpy as np
import pytest
import torch

from nemotron_infer_amd import _lib, ops
from oracle import block, paged
from tests.gpu_util import DEV, announce, assert_parity, bits
from tests.test_paged_gpu import Pool, _dev, _f64, _rand_bits

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _no_pending_error():
    _lib.lib().nmi_async_status()
    yield
    torch.cuda.synchronize()
    _lib.lib().nmi_async_status()


def _selected(pool, q, bounds, select):
    """(o, places) of one call."""
    places = torch.full((len(pool.lens), pool.k.shape[1], select), -7, dtype=torch.int32, device=DEV)
    o = ops.sdpa_decode_paged_sparse(_dev(q), pool.dk, pool.dv, pool.dtable, _dev(pool.lens), _dev(bounds), select, selected=places)
    torch.cuda.synchronize()
    assert _lib.lib().nmi_async_status() == 0
    return o, places.cpu().numpy()


LARGEST = (2.0 - 2.0 ** -7) * 2.0 ** 127


@pytest.mark.parametrize("far", [2.0 ** 20, 2.0 ** 36, 2.0 ** 50, 2.0 ** 60, 2.0 ** 100, LARGEST])
@pytest.mark.parametrize("H,n_kv", [(1, 1), (2, 1), (8, 2), (5, 1), (7, 1)])
def test_scores_take_nothing_from_the_side_that_no_query_uses(far, H, n_kv):
    """A dim whose queries are all negative and whose largest key is far out, another the other way round: the score is the
    other dims' and the near side's."""
    announce("sparse_one_sided", far, H, n_kv)
    rng = np.random.default_rng(H)
    pool = Pool(rng, [1500, 700], n_kv, 16, "bf16")
    q = _f64(_rand_bits(rng, 2, H * 128)).reshape(2, H, 128)
    q[:, :, 40], q[:, :, 77] = -np.abs(q[:, :, 40]), np.abs(q[:, :, 77])
    x = np.sort(rng.standard_normal((pool.k.shape[0], n_kv, 2, 128)), axis=2)
    some = rng.random((pool.k.shape[0], n_kv)) < 0.7
    x[..., 1, 40] = np.where(some, far, x[..., 1, 40])
    x[..., 0, 77] = np.where(~some, -far, x[..., 0, 77])
    q, bounds = block.bf16_round_exact(q), block.bf16_round_exact(x)
    o, places = _selected(pool, q.reshape(2, -1), bounds, 12)
    kept = [paged.select(_f64(q[b]), _f64(bounds), pool.table[b], int(n), 16, 12) for b, n in enumerate(pool.lens)]
    assert np.array_equal(places, kept)
    want = paged.decode_selected(_f64(q), *pool.values(), pool.table, pool.lens, kept)
    assert_parity(bits(o).reshape(want.shape), block.bf16_round_exact(want), f"{far}", per_row_scales=True)


@pytest.mark.parametrize("sign", [1, -1])
def test_an_infinite_query_scores_infinities(sign):
    """+inf * hi where hi > 0 is the largest score, where hi < 0 the smallest, whatever lo is (0 * lo = 0); so with the signs
    turned."""
    announce("sparse_infinite", sign)
    rng = np.random.default_rng(5)
    pool = Pool(rng, [640], 1, 16, "bf16")
    q = _f64(_rand_bits(rng, 1, 128))
    q[0, 9] = sign * np.inf
    x = np.sort(rng.standard_normal((pool.k.shape[0], 1, 2, 128)), axis=2)
    first = [3, 11, 12, 38]
    used, other = (1, 0) if sign > 0 else (0, 1)
    x[:, 0, used, 9], x[:, 0, other, 9] = -sign, -4.0 * sign if sign > 0 else 4.0
    x[pool.table[0, first], 0, used, 9] = sign
    _, places = _selected(pool, block.bf16_round_exact(q), block.bf16_round_exact(x), 5)
    assert places.tolist() == [[first + [39]]]


def test_the_newest_page_alone_needs_no_scores():
    """n_select 1: places of pages that nothing could score are left as they were, page ids out of range there are not
    met, and the newest page is attended."""
    announce("sparse_newest")
    rng = np.random.default_rng(6)
    lens = [777, 3000, 16, 0]
    pool = Pool(rng, lens, 2, 16, "bf16")
    q, bounds = _rand_bits(rng, 4, 8 * 128), _rand_bits(rng, pool.k.shape[0], 2, 2, 128)
    pool.table[0, 5], pool.table[1, 0] = -1, pool.k.shape[0]
    width, L = pool.table.shape[1], _lib.lib()
    dk, dv, dtable, dlens, dq, dbounds = pool.dk, pool.dv, _dev(pool.table), _dev(pool.lens), _dev(q), _dev(bounds)
    c = _lib.PagedKv(dk.data_ptr(), dv.data_ptr(), 2 * 16 * 128, 16 * 128, 128, dtable.data_ptr(), width, None, None, 0,
                     dk.shape[0], 16, width, 2)
    ws = torch.full((L.nmi_sdpa_decode_paged_sparse_workspace_bytes(4, 8, 2, width, 1),), 0x5A, dtype=torch.uint8, device=DEV)
    o = torch.empty(4, 8 * 128, dtype=torch.bfloat16, device=DEV)
    places = torch.empty(4, 2, 1, dtype=torch.int32, device=DEV)
    rc = L.nmi_sdpa_decode_paged_sparse(ctypes.addressof(c), dq.data_ptr(), 8 * 128, o.data_ptr(), 8 * 128, dlens.data_ptr(),
                                        dbounds.data_ptr(), 1, places.data_ptr(), 4, 8, 128 ** -0.5, ws.data_ptr(), ws.numel(),
                                        torch.cuda.current_stream().cuda_stream)
    assert rc == 0, L.nmi_last_error()
    torch.cuda.synchronize()
    assert L.nmi_async_status() == 0
    assert places.tolist() == [[[48]] * 2, [[187]] * 2, [[0]] * 2, [[-1]] * 2]
    assert (ws[:4 * 2 * width * 4] == 0x5A).all()                                 # (the scores)
    kept = [[[48]] * 2, [[187]] * 2, [[0]] * 2, [[]] * 2]
    want = paged.decode_selected(_f64(q).reshape(4, 8, 128), *pool.values(), pool.table, pool.lens, kept)
    assert_parity(bits(o)[:3].reshape(3, 8, 128), block.bf16_round_exact(want[:3]), "newest", per_row_scales=True)
    assert not bits(o)[3].any()


@pytest.mark.parametrize("batch,width,page", [(40, 1024, 1 << 20), (300, 3000, 16)])
def test_pages_past_the_stack_are_neither_pushed_nor_read(batch, width, page):
    """Ended sequences whose lengths claim many times the pool's pages: the stack is filled in the sequences' order, the rest
    dropped, and reported once; ids behind those that fit, out of range here, are not met."""
    announce("assign_claims", batch, width, page)
    n_pages, count = 50, 20
    table = torch.full((batch, width), -9, dtype=torch.int32, device=DEV)
    table[0, :30] = torch.arange(20, 50)
    lens = torch.full((batch,), width * page, dtype=torch.int32, device=DEV)
    free = torch.arange(n_pages, dtype=torch.int32, device=DEV)
    free[count:] = -5
    new = torch.full((batch,), -1, dtype=torch.int32, device=DEV)
    got = ops.kv_assign_paged(lens, new, table, free, torch.tensor([count], dtype=torch.int32, device=DEV), page, tokens=0)
    torch.cuda.synchronize()
    assert _lib.lib().nmi_async_status() == _lib.NMI_ERR_ASYNC and _lib.lib().nmi_async_status() == 0
    assert got.free_count.tolist() == [n_pages] and free.tolist() == list(range(n_pages))
    assert (got.lens == -1).all() and (got.start_pos == -1).all() and (table[:, 30:] == -9).all()


def test_a_shared_prefix_outlives_the_sequence_that_ends_first():
    """Two sequences share the full pages of a prefix and grow here; the first is ended by hand (its own pages on the stack,
    its length negative), the last one here.  At each step every page is free, or held by those that share it."""
    announce("assign_shared")
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)  # noqa: E731
    page, shared = 16, [7, 3]
    table, lens = ints([[7, 3, 1, -1, -1], [7, 3, -1, -1, -1], [-1] * 5]), ints([40, 32, -1])
    free, count = ints([0, 2, 4, 5, 6, -1, -1, -1]), ints([5])

    def step(*new):
        got = ops.kv_assign_paged(lens, ints(list(new)), table, free, count, page, tokens=sum(max(0, n) for n in new),
                                  lens_out=lens, free_count_out=count)
        torch.cuda.synchronize()
        assert _lib.lib().nmi_async_status() == 0
        rows = [table[b, :-(-max(0, int(n)) // page)].tolist() for b, n in enumerate(lens)]
        held = {i for r in rows for i in r}
        own = [i for r in rows for i in r if i not in shared]
        assert len(own) == len(set(own)) and sorted([*held, *free[:int(count)].tolist()]) == list(range(8))
        return got, rows

    got, rows = step(10, 5, 0)
    assert got.lens.tolist() == [50, 37, -1] and rows == [[7, 3, 1, 6], [7, 3, 5], []]
    c, own = int(count), table[0, 2:4]
    free[c:c + own.numel()] = own
    count += own.numel()
    lens[0] = -1
    lens[2] = 0
    got, rows = step(0, 13, 33)
    assert got.start_pos.tolist() == [-1, 37, 0] and rows == [[], [7, 3, 5, 6], [1, 4, 2]]
    got, rows = step(0, -1, 1)
    assert rows == [[], [], [1, 4, 2]] and free[:int(count)].tolist() == [0, 7, 3, 5, 6]


@pytest.mark.parametrize("batch", [1, 3])
def test_entries_past_a_sequences_pages_change_nothing(batch):
    """A table far wider than the sequences, its unused entries naming pages that others hold, whose bounds would be chosen
    first, or no pages: the same bytes as with a table just wide enough."""
    announce("sparse_wide", batch)
    rng = np.random.default_rng(batch)
    lens = [1000, 333, 530][:batch]
    pool = Pool(rng, lens, 2, 16, "bf16", extra=40)
    q = _rand_bits(rng, batch, 8 * 128)
    x = np.sort(rng.standard_normal((pool.k.shape[0], 2, 2, 128)), axis=2)
    idle = np.setdiff1d(np.arange(len(x)), pool.table)
    x[idle[::2]], x[idle[1::2]] = np.nan, np.inf
    bounds = block.bf16_round_exact(x)
    o, places = _selected(pool, q, bounds, 7)
    wide = np.full((batch, 4000), 2 ** 31 - 1, np.int32)
    wide[:, :1500] = rng.choice(idle, (batch, 1500))
    for b, n in enumerate(lens):
        used = -(-n // 16)
        wide[b, :used] = pool.table[b, :used]
    pool.dtable = _dev(wide)
    again, places_again = _selected(pool, q, bounds, 7)
    assert np.array_equal(places, places_again) and np.array_equal(bits(o), bits(again))
