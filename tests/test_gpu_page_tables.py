"""Page tables and slot maps from the requests' lengths, and accepted paths moved in the pages, on the device against their
definitions a request at a time. All whole numbers and copies: equal."""
import numpy as np
import pytest

import aqueduct as aq
import paged_plain as P
import tree_plain as T

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    return aq.Context(0)


class Device:
    """A pool's tables on the device beside the definition's."""

    def __init__(self, ctx, n_seq, max_pages, n_pages, page, rng, in_place=True):
        self.ctx, self.want, self.in_place = ctx, T.Tables(n_seq, max_pages, n_pages, page), in_place
        w = self.want
        w.ring = rng.permutation(n_pages).astype(np.int32)
        w.first = int(rng.integers(0, n_pages))
        self.pages, self.held, self.ring = P.Dev(ctx, w.pages), P.Dev(ctx, w.held), P.Dev(ctx, w.ring)
        self.state = P.Dev(ctx, np.array([w.first, w.count, 0, 0], np.int32))
        self.held_out, self.state_out = P.Dev(ctx, w.held), P.Dev(ctx, np.zeros(4, np.int32))
        out = {} if in_place else dict(held_out=self.held_out.buf, free_state_out=self.state_out.buf)
        self.t = aq.page_tables(n_seq, max_pages, n_pages, page, self.pages.buf, self.held.buf, self.ring.buf,
                                self.state.buf, **out)

    def call(self, before, new, n_rows, depth=None, in_place_len=False, stream=None):
        ctx, n = self.ctx, self.want.n_seq
        self.d = {"before": P.Dev(ctx, np.array(before, np.int32)), "new": P.Dev(ctx, np.array(new, np.int32)),
                  "start": P.Dev(ctx, np.full(n + 1, 5, np.int32)), "len": P.Dev(ctx, np.full(n, 5, np.int32)),
                  "missing": P.Dev(ctx, np.full(n, 5, np.int32)), "pos": P.Dev(ctx, np.full(n_rows + 3, 5, np.int32)),
                  "slots": P.Dev(ctx, np.full(n_rows + 3, 5, np.int64)),
                  "depth": None if depth is None else P.Dev(ctx, np.array(depth, np.int32))}
        d = self.d
        if in_place_len:
            d["len"] = d["before"]
        aq.paged_tables(ctx, self.t, d["before"].buf, d["new"].buf, n_rows, d["start"].buf, d["len"].buf, d["missing"].buf,
                        d["pos"].buf, d["slots"].buf, None if depth is None else d["depth"].buf, stream=stream)

    def check(self, before, new, n_rows, depth=None, times=1, **kw):
        for _ in range(times):
            self.call(before, new, n_rows, depth, **kw)
            self.ctx.sync()
        w = self.want
        want = dict(zip(("start", "len", "missing", "pos", "slots"), w.step(before, new, n_rows, depth)))
        for name, x in want.items():
            got = self.d[name].get()
            assert np.array_equal(got[: len(x)], x), (name, np.nonzero(got[: len(x)] != x)[0][:5])
            assert np.all(got[len(x):] == 5)
        held, state = (self.held, self.state) if self.in_place else (self.held_out, self.state_out)
        assert np.array_equal(held.get(), w.held)
        assert state.get().tolist() == [w.first, w.count, 0, 0]
        assert np.array_equal(self.pages.get(), w.pages) and np.array_equal(self.ring.get(), w.ring)
        if not self.in_place:
            self.held.buf.upload(w.held)
            self.state.buf.upload(np.array([w.first, w.count, 0, 0], np.int32))
        return want


@pytest.mark.parametrize("in_place", [True, False])
@pytest.mark.parametrize("n_seq,page,pool,most", [(1, 16, 40, 30), (5, 1, 200, 20), (48, 16, 400, 3), (300, 7, 900, 90),
                                                  (1024, 4, 3000, 9), (1025, 16, 1500, 40), (2500, 3, 9000, 6), (64, 64, 64, 900)])
def test_steps(ctx, in_place, n_seq, page, pool, most):
    """Requests that begin, grow, end and start again over steps; pools that run out now and then."""
    print(f"tables {n_seq} page {page} pool {pool} most {most} in place {in_place}", flush=True)
    rng = np.random.default_rng(n_seq + page)
    dev = Device(ctx, n_seq, max(2, 2 * most // page), pool, page, rng, in_place)
    lens = np.zeros(n_seq, np.int64)
    for step in range(6):
        new = rng.integers(0, most + 1, n_seq)
        new[rng.random(n_seq) < 0.2] = -1
        new[rng.random(n_seq) < 0.1] = 0
        rows = int(np.maximum(new, 0).sum())
        n_rows = rows + int(rng.integers(-min(rows, 5), 9))
        depth = rng.integers(0, 9, n_rows) if step % 2 else None
        want = dev.check(lens, new, n_rows, depth, times=1 if in_place else 2, in_place_len=in_place and step == 3)
        # a sequence whose pages ran out, or whose table is full, goes on with what it has; drafts are dropped now and then
        lens = np.where(want["missing"] > 0, np.minimum(lens * (new >= 0), dev.want.held * page), want["len"])
        lens = np.maximum(lens - rng.integers(0, 3, n_seq), 0)


@pytest.mark.parametrize("n_seq", [3, 2000])
def test_extremes(ctx, n_seq):
    """Lengths below 0, sums past 31 bits, counts that no table holds, garbage in the tables and the ring: every access in
    range, lengths saturated, and no slot outside the pool."""
    print(f"extremes {n_seq}", flush=True)
    rng = np.random.default_rng(1)
    dev = Device(ctx, n_seq, 5, 50, 8, rng)
    before, new = np.zeros(n_seq, np.int64), np.zeros(n_seq, np.int64)
    before[:3], new[:3] = [2 ** 31 - 1, -9, 2 ** 31 - 5], [2 ** 31 - 1, 4, 7]
    dev.call(before, new, 300)
    ctx.sync()
    assert dev.d["len"].get()[:3].tolist() == [2 ** 31 - 1, 4, 2 ** 31 - 1]
    assert dev.d["start"].get()[:3].tolist() == [0, 2 ** 31 - 1, 2 ** 31 - 1]
    assert np.all(dev.d["slots"].get()[:300] == -1)
    assert dev.d["missing"].get()[0] == 2 ** 28 - 5 and dev.held.get()[0] == 5
    dev.held.buf.upload(rng.integers(-2 ** 31, 2 ** 31, n_seq).astype(np.int32))
    dev.state.buf.upload(np.array([-7, 2 ** 31 - 1, 0, 0], np.int32))
    dev.ring.buf.upload(rng.integers(-2 ** 31, 2 ** 31, 50).astype(np.int32))
    dev.call(rng.integers(-50, 50, n_seq), rng.integers(-1, 40, n_seq), 5000)
    ctx.sync()
    slots, state = dev.d["slots"].get()[:5000], dev.state.get()
    assert np.all((slots >= -1) & (slots < 400)) and 0 <= state[0] < 50 and 0 <= state[1] <= 50 and state[2] == 0


def test_nothing(ctx):
    """No sequence: row_start is 0, every row is behind the last; null outputs are left out."""
    dev = Device(ctx, 1, 4, 9, 16, np.random.default_rng(2))
    t = aq.page_tables(0, 4, 9, 16, dev.pages.buf, dev.held.buf, dev.ring.buf, dev.state.buf)
    start, slots = P.Dev(ctx, np.full(1, 5, np.int32)), P.Dev(ctx, np.full(4, 5, np.int64))
    aq.paged_tables(ctx, t, dev.held.buf, dev.held.buf, 3, start.buf, dev.held_out.buf, slots=slots.buf)
    ctx.sync()
    assert start.get().tolist() == [0] and slots.get().tolist() == [-1, -1, -1, 5]
    assert dev.state.get().tolist() == [dev.want.first, 9, 0, 0]


# -------------------------------------------------------------------------------------------------- accepted paths
def committed(pg, paths, m):
    """(K, V, lengths) after the paths: by the definition, position by position."""
    k, v, lens = pg.k.copy(), pg.v.copy(), []
    for s, (n, length) in enumerate(zip(pg.new, pg.lens)):
        base = max(length, 0) - n
        kept = 0
        for i in range(min(max(int(m[s]), 0), paths.shape[1])):
            j = int(paths[s, i])
            if not 0 <= j < n or (i and j <= paths[s, i - 1]):
                break
            kept += 1
            a, b = pg.row_of(s, base + j), pg.row_of(s, base + i)
            if a is not None and b is not None:
                k[b], v[b] = k[a], v[a]
        lens.append(max(base + kept, 0))
    return k, v, lens


@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("kv,hd,page,layout", [(2, 64, 16, "slots"), (4, 256, 7, "heads"), (1, 8, 1, "slots"), (16, 80, 64, "slots"),
                                               (33, 256, 16, "slots")])
@pytest.mark.parametrize("layers", [1, 3])
def test_commit(ctx, t, kv, hd, page, layout, layers):
    print(f"commit {t} {kv} x {hd} page {page} {layout} layers {layers}", flush=True)
    rng = np.random.default_rng(kv + hd)
    new = [26, 1, 0, 150, 9, 12, 5, 30]
    lens = [40, 30, 9, 150, 200, 5, -3, 90]  # one shorter than its new rows
    most = 100
    first = P.Paged(ctx, rng, new, lens, kv, hd, page, t, layout=layout)
    pgs = [first]
    for _ in range(layers - 1):  # the same tables, other rows
        pg = P.Paged.__new__(P.Paged)
        pg.__dict__.update(first.__dict__)
        pg.k, pg.v = rng.standard_normal(first.k.shape), rng.standard_normal(first.v.shape)
        pgs.append(pg)
    first.table[7, 70 // page] = -1  # a hole inside the tree
    for pg in pgs:
        pg.upload()
    paths, m = np.full((8, most), -1, np.int32), np.zeros(8, np.int32)
    for s, n in enumerate(new):
        c = int(rng.integers(1, n + 1)) if n else 3
        c = 90 if n == 150 else c
        path = np.sort(rng.choice(max(n, 3), min(c, max(n, 3)), replace=False))
        paths[s, : len(path)], m[s] = path, len(path)
    m[1], m[4] = 1000, -1       # more than the path has room for; none
    paths[5, :6] = [0, 2, 4, 4, 5, 6]  # stops rising
    paths[7, :6], m[7] = [1, 3, 5, 29, 30, 31], 6  # leaves the tree
    want = [committed(pg, paths, m) for pg in pgs]
    dp, dm, out = P.Dev(ctx, paths), P.Dev(ctx, m), P.Dev(ctx, np.full(8, 5, np.int32))
    caches = aq.paged_kv_array([pg.structs()[0] for pg in pgs])
    aq.paged_tree_commit(ctx, caches, pgs[0].structs()[1], dp.buf, dm.buf, most, out.buf)
    ctx.sync()
    for pg, (k, v, length) in zip(pgs, want):
        got = pg.pools()
        assert np.array_equal(got[0], k, equal_nan=True) and np.array_equal(got[1], v, equal_nan=True)
        assert out.get().tolist() == length


def test_commit_of_many_caches(ctx):
    """More caches than one launch has; without lengths."""
    print("commit of 130 caches", flush=True)
    rng = np.random.default_rng(5)
    pgs = [P.Paged(ctx, np.random.default_rng(9), [8, 3], [20, 30], 2, 16, 16, "f16") for _ in range(130)]
    for pg in pgs:
        pg.k, pg.v = rng.standard_normal(pg.k.shape), rng.standard_normal(pg.v.shape)
        pg.upload()
    paths, m = np.array([[0, 3, 7], [1, 2, -1]], np.int32), np.array([3, 2], np.int32)
    dp, dm = P.Dev(ctx, paths), P.Dev(ctx, m)
    aq.paged_tree_commit(ctx, aq.paged_kv_array([pg.structs()[0] for pg in pgs]), pgs[0].structs()[1], dp.buf, dm.buf, 3)
    ctx.sync()
    for pg in pgs:
        k, v, _ = committed(pg, paths, m)
        got = pg.pools()
        assert np.array_equal(got[0], k) and np.array_equal(got[1], v)
