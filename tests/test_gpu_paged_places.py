"""Which rows of the row tensors and which positions of the cache the paged calls touch: sequences that begin past the
tensor's first row or before it, or end past its last; lengths below 0; queries of rows without a page. Append and attention
place a row alike. Tolerances: paged_plain.bound and rotate_bound; what is not a row's stays bit for bit."""
import numpy as np
import pytest

import aqueduct as aq
import paged_plain as P
from test_gpu_paged_attention import PAIRS, bounds, run

pytestmark = pytest.mark.gpu
THETA = 1e6


@pytest.fixture(scope="module")
def ctx():
    return aq.Context(0)


class Shifted:
    """A batch whose row_start begins at `first`, over row tensors of n rows: sequence s's row i is row
    first + (rows before it) + i of the tensors, or none of them."""

    def __init__(self, ctx, rng, new, lens, first, n, kv, hd, cache_t, page=16):
        self.pg = P.Paged(ctx, rng, new, lens, kv, hd, page, cache_t, n_rows=n)
        self.first, self.n = first, n
        self.pg.dstarts = P.Dev(ctx, (self.pg.starts + first).astype(np.int32))
        self.rows = [(int(self.pg.starts[s]) + first + i, s, max(lens[s], 0) - a + i)
                     for s, a in enumerate(new) for i in range(a)]
        self.rows = [(r, s, p) for r, s, p in self.rows if 0 <= r < n]
        self.mine = np.zeros(n, bool)
        self.mine[[r for r, _, _ in self.rows]] = True

    def attention(self, q, scale, window=0):
        """The definition's outputs and its bound's parts, of the tensors' rows."""
        lead = max(0, -self.first)
        wide = np.concatenate([np.zeros((lead, *q.shape[1:])), q])
        plain = P.Paged.__new__(P.Paged)
        plain.__dict__.update(self.pg.__dict__, starts=self.pg.starts + self.first + lead)
        want, parts = P.attention(plain, wide, scale, window)
        return want[lead:], tuple(x[lead:] for x in parts)


@pytest.mark.parametrize("row_t,cache_t", PAIRS)
@pytest.mark.parametrize("first,cut", [(5, 0), (0, 1), (7, 2), (-1, 0), (-2, 1)])
@pytest.mark.parametrize("new", [[2, 4, 4], [40, 0, 45, 40], [1] * 70])
@pytest.mark.parametrize("window", [0, 30])
def test_attention_of_rows_around_the_tensor(ctx, row_t, cache_t, first, cut, new, window):
    """Rows before the first sequence and rows that the tensors do not have; a sequence that is cut keeps its other rows'
    positions."""
    print(f"places {row_t}/{cache_t} first {first} cut {cut} new {new[:4]} x {len(new)} window {window}", flush=True)
    rng = np.random.default_rng(61)
    lens = [n + int(x) for n, x in zip(new, rng.integers(0, 300, len(new)))]
    n = first + sum(new) - cut
    b = Shifted(ctx, rng, new, lens, first, n, 2, 64, cache_t)
    q = P.Rows(ctx, rng.standard_normal((n, 4, 64)), row_t)
    want, parts = b.attention(q.values(), 0.125, window)
    limit = P.bound(parts, want, row_t, cache_t, 64)
    for loose in bounds(b.pg, q):
        out = P.Rows(ctx, np.full((n, 4, 64), 9.0), row_t)
        run(ctx, b.pg, q, out, 0.125, window, loose=loose)
        got = out.get()
        assert np.all(got[~b.mine] == 9.0)
        assert np.all(np.abs(got - want)[b.mine] <= limit[b.mine])


@pytest.mark.parametrize("row_t,cache_t", PAIRS)
@pytest.mark.parametrize("first,cut", [(0, 0), (5, 0), (0, 1), (7, 2), (-1, 0), (-2, 1)])
@pytest.mark.parametrize("new", [[2, 4, 4], [40, 0, 45, 40], [1] * 70])
@pytest.mark.parametrize("in_place", [False, True])
def test_append_of_rows_around_the_tensor(ctx, row_t, cache_t, first, cut, new, in_place):
    """Only the sequences' rows are stored, at the positions that attention gives them, and only their queries turned: the
    rows before the first start are somebody else's, and what the cache held stays."""
    print(f"places, append {row_t}/{cache_t} first {first} cut {cut} new {new[:4]} x {len(new)} in place {in_place}", flush=True)
    rng = np.random.default_rng(62)
    lens = [n + int(x) for n, x in zip(new, rng.integers(0, 300, len(new)))]
    lens[0] = 103 + new[0]
    n = first + sum(new) - cut
    b = Shifted(ctx, rng, new, lens, first, n, 2, 64, cache_t)
    check_append(ctx, rng, b, row_t, cache_t, in_place)


@pytest.mark.parametrize("row_t,cache_t", PAIRS)
@pytest.mark.parametrize("below", [-1, -5, -2 ** 31 + 1])
def test_append_at_lengths_below_zero(ctx, row_t, cache_t, below):
    """A length below 0 counts as 0: the rows stand before position 0, store nothing, and are turned by where they stand."""
    print(f"places, length {below} {row_t}/{cache_t}", flush=True)
    rng = np.random.default_rng(63)
    b = Shifted(ctx, rng, [3, 2, 1], [below, 40, 0], 0, 6, 2, 64, cache_t)
    check_append(ctx, rng, b, row_t, cache_t, False)


def check_append(ctx, rng, b, row_t, cache_t, in_place):
    pg, n = b.pg, b.n
    k, v = (P.Rows(ctx, rng.standard_normal((n, 2, 64)), row_t) for _ in range(2))
    q = P.Rows(ctx, rng.standard_normal((n, 4, 64)), row_t)
    qo = q if in_place else P.Rows(ctx, np.full((n, 4, 64), 9.0), row_t)
    cache, batch = pg.structs()
    rope = aq.Rope(ctx, 48, THETA)
    aq.paged_append(ctx, cache, batch, k.heads_struct(), v.heads_struct(), rope, q.heads_struct(), qo.heads_struct(), 4)
    ctx.sync()
    pos = np.zeros(n, np.int64)
    for r, _, p in b.rows:
        pos[r] = p
    freq, _ = P.frequencies(48, THETA)
    turned_k, turned_q = (P.rotate(x.values(), pos, 48, "half", freq) for x in (k, q))
    limit = P.rotate_bound(k.values(), turned_k, cache_t)
    got_k, got_v = pg.pools()
    want_k, want_v = pg.k.copy(), pg.v.copy()
    for r, s, p in b.rows:
        at = pg.row_of(s, p)
        if at is None:
            continue
        assert np.all(np.abs(got_k[at] - turned_k[r]) <= limit[r]), (r, s, p)
        want_k[at], want_v[at] = got_k[at], P.values(P.store(v.values()[r], cache_t), cache_t)
    assert np.array_equal(want_k, got_k, equal_nan=True), "keys that are not the rows'"
    assert np.array_equal(want_v, got_v, equal_nan=True), "values that are not the rows'"
    got, before = qo.get(), q.values() if in_place else np.full((n, 4, 64), 9.0)
    assert np.array_equal(got[~b.mine], before[~b.mine]), "queries of rows that are no sequence's"
    assert np.all((np.abs(got - turned_q) <= P.rotate_bound(q.values(), turned_q, row_t))[b.mine])


@pytest.mark.parametrize("row_t,cache_t", PAIRS)
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("in_place", [False, True])
def test_queries_of_rows_without_a_page_are_turned(ctx, row_t, cache_t, layout, in_place):
    """At negative positions, in holes and past the table a row stores nothing; its q is rotated all the same."""
    rng = np.random.default_rng(64)
    pg = P.Paged(ctx, rng, [4, 3, 2], [2, 60, 40], 2, 64, 16, cache_t, cols=3)
    pg.table[2, 2] = pg.k.shape[0]  # positions 32 .. 47; those of sequence 1 lie past the table
    pg.upload()
    k = P.Rows(ctx, rng.standard_normal((9, 2, 64)), row_t)
    q = P.Rows(ctx, rng.standard_normal((9, 4, 64)), row_t)
    qo = q if in_place else P.Rows(ctx, np.full((9, 4, 64), 9.0), row_t)
    cache, batch = pg.structs()
    aq.paged_append(ctx, cache, batch, k.heads_struct(), k.heads_struct(), aq.Rope(ctx, 64, THETA, layout=layout),
                    q.heads_struct(), qo.heads_struct(), 4)
    ctx.sync()
    pos = np.array([-2, -1, 0, 1, 57, 58, 59, 38, 39])
    want = P.rotate(q.values(), pos, 64, layout, P.frequencies(64, THETA)[0])
    assert np.all(np.abs(qo.get() - want) <= P.rotate_bound(q.values(), want, row_t))
    want_v = pg.v.copy()
    for r in (2, 3):
        want_v[pg.row_of(0, int(pos[r]))] = P.values(P.store(k.values()[r], cache_t), cache_t)
    assert np.array_equal(want_v, pg.pools()[1], equal_nan=True)
