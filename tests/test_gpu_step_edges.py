"""The calls of a speculative step over pages where their arguments end: heads that leave lanes of a wave without one, trees
that begin before the row tensors, mask words longer than a tree, rows of any number of pieces to move, more work-groups
than one dimension has, a pool that runs out. Against the definitions, in 64 bits; tolerances: tree_plain.norm_bound and
paged_plain.bound, by arithmetic; what is copied is equal."""
import math

import numpy as np
import pytest

import aqueduct as aq
import paged_plain as P
import tree_plain as T

pytestmark = pytest.mark.gpu
PAIRS = [("f32", "f32"), ("f32", "f16"), ("f32", "bf16"), ("f16", "f16"), ("bf16", "bf16")]
THETA, EPS = 1e6, 1e-6


@pytest.fixture(scope="module")
def ctx():
    return aq.Context(0)


@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("hd,dim,pad", [(8, 8, 0), (16, 8, 0), (64, 32, 0), (128, 128, 0), (256, 64, 0), (96, 48, 1), (10, 4, 1)])
def test_one_tensor_of_any_number_of_heads(ctx, t, layout, hd, dim, pad):
    """Queries alone and keys alone, the other's weight null: each number of heads leaves other lanes without one."""
    rng = np.random.default_rng(hd)
    rope = aq.Rope(ctx, dim, THETA, layout=layout)
    freq, gain = P.frequencies(dim, THETA)
    for heads in (1, 2, 3, 5, 17, 63, 65):
        print(f"one tensor {t} {layout} {heads} x {hd} of {dim} pad {pad}", flush=True)
        x = P.Rows(ctx, rng.standard_normal((3, heads, hd)) * 2, t, pad)
        w = (1 + 0.3 * rng.standard_normal(hd)).astype(np.float32)
        pos = rng.integers(0, 9000, 3).astype(np.int32)
        dw, dpos = P.Dev(ctx, w), P.Dev(ctx, pos)
        want = P.rotate(T.normed(x.values(), w.astype(np.float64), EPS), pos, dim, layout, freq, gain)
        limit = T.norm_bound(x.values(), w.astype(np.float64), EPS, want, t, dim, gain)
        for first in (True, False):
            out = P.Rows(ctx, np.full((3, heads, hd), 9.0), t, pad)
            one, none = (x.heads_struct(), out.heads_struct(), heads), (None, None, 0)
            aq.qk_norm_rope(ctx, *(one if first else none), *(none if first else one), hd, 3, dw.buf if first else None,
                            None if first else dw.buf, EPS, rope, dpos.buf)
            ctx.sync()
            assert np.all(np.abs(out.get() - want) <= limit)


@pytest.mark.parametrize("row_t,cache_t", PAIRS)
@pytest.mark.parametrize("new,window", [(7, 0), (7, 9), (70, 0), (70, 90)])
def test_trees_that_begin_before_the_tensors(ctx, row_t, cache_t, new, window):
    """row_start below 0: the rows that there are have their own masks, whose bits count from the tree's first row."""
    print(f"begins before {row_t}/{cache_t} new {new} window {window}", flush=True)
    rng = np.random.default_rng(new)
    heads, kv, hd, skip = 4, 2, 128, new // 2 + 1
    pg = P.Paged(ctx, rng, [new, 5], [new + 200, 77], kv, hd, 16, cache_t)
    masks = [m | (rng.random(len(m)) < 0.3) for m in T.random_trees(rng, pg.new)]
    x = rng.standard_normal((pg.rows, heads, hd))
    scale = float(np.float32(1.0 / math.sqrt(hd)))
    want, parts = T.tree_attention(pg, masks, P.values(P.store(x, row_t), row_t), scale, window)
    limit = P.bound(parts, want, row_t, cache_t, hd)[skip:]
    q, out = P.Rows(ctx, x[skip:], row_t), P.Rows(ctx, np.full(x[skip:].shape, 9.0), row_t)
    starts, words = P.Dev(ctx, (pg.starts - skip).astype(np.int32)), -(-new // 32)
    dm = P.Dev(ctx, T.pack(masks[skip:], words))
    cache, _ = pg.structs()
    for most in (pg.max_len, 5 << 20):  # the second: bounds with which many 16-bit rows take a kernel of their own
        table = np.full((2, -(-max(most, 300) // 16)), -1, np.int32)
        table[:, : pg.cols] = pg.table
        dt = P.Dev(ctx, table)
        b = aq.paged_batch(2, starts.buf, pg.dlens.buf, dt.buf, table.shape[1], q.rows, new, most)
        ws = aq.DeviceBuffer(ctx, aq.paged_attention_workspace(ctx, cache, b, heads))
        aq.paged_tree_attention(ctx, cache, b, dm.buf, words, heads, q.heads_struct(), out.heads_struct(), scale, window, None, ws)
        ctx.sync()
        assert np.all(np.abs(out.get() - want[skip:]) <= limit)


def test_paths_of_trees_that_begin_before_the_tensors(ctx):
    """The rows to move lie in the pages, wherever the row tensors begin: of one that begins before them, of one that ends
    before them, and of one that ends past them."""
    rng = np.random.default_rng(3)
    pg = P.Paged(ctx, rng, [4, 9, 6], [30, 50, 21], 2, 64, 16, "bf16")
    paths, m = np.array([[1, 3, -1, -1], [0, 2, 5, 8], [2, 3, 5, -1]], np.int32), np.array([2, 4, 3], np.int32)
    starts, dp, dm = P.Dev(ctx, pg.starts - 7), P.Dev(ctx, paths), P.Dev(ctx, m)
    out = P.Dev(ctx, np.full(3, 5, np.int32))
    cache, _ = pg.structs()
    b = aq.paged_batch(3, starts.buf, pg.dlens.buf, pg.dtable.buf, pg.cols, 9, 9, 50)
    aq.paged_tree_commit(ctx, aq.paged_kv_array([cache]), b, dp.buf, dm.buf, 4, out.buf)
    ctx.sync()
    k, v = pg.k.copy(), pg.v.copy()
    for s in range(3):
        base = pg.lens[s] - pg.new[s]
        for i in range(int(m[s])):
            a, to = pg.row_of(s, base + int(paths[s, i])), pg.row_of(s, base + i)
            k[to], v[to] = k[a], v[a]
    got = pg.pools()
    assert np.array_equal(got[0], k, equal_nan=True) and np.array_equal(got[1], v, equal_nan=True)
    assert out.get().tolist() == [n - w + int(x) for n, w, x in zip(pg.lens, pg.new, m)]


@pytest.mark.parametrize("row_t,cache_t", PAIRS)
@pytest.mark.parametrize("n", [1, 5, 31, 32, 33])
def test_bits_past_a_short_tree(ctx, row_t, cache_t, n):
    """Beside a large tree a small one whose words hold ones past its own rows: with a window they count for nothing."""
    print(f"spare bits {row_t}/{cache_t} {n}", flush=True)
    rng = np.random.default_rng(n)
    heads, kv, hd, big, words = 4, 2, 64, 70, 4
    pg = P.Paged(ctx, rng, [n, big, n], [n + 100, big + 60, n + 3], kv, hd, 16, cache_t)
    masks = T.random_trees(rng, pg.new)
    packed = T.pack(masks, words)
    for r, m in enumerate(masks):
        spare = np.ones(32 * words, bool)
        spare[: len(m)] = False
        packed[r] |= T.pack([spare], words)[0]
    dm = P.Dev(ctx, packed)
    q = P.Rows(ctx, rng.standard_normal((pg.rows, heads, hd)), row_t)
    scale = float(np.float32(1.0 / math.sqrt(hd)))
    for window in (1, 40, 140):
        want, parts = T.tree_attention(pg, masks, q.values(), scale, window)
        limit = P.bound(parts, want, row_t, cache_t, hd)
        for most in (pg.max_len, 5 << 16):
            table = np.full((3, -(-most // 16)), -1, np.int32)
            table[:, : pg.cols] = pg.table[:, : table.shape[1]]
            dt = P.Dev(ctx, table)
            cache, _ = pg.structs()
            b = aq.paged_batch(3, pg.dstarts.buf, pg.dlens.buf, dt.buf, table.shape[1], pg.rows, big, most)
            ws = aq.DeviceBuffer(ctx, aq.paged_attention_workspace(ctx, cache, b, heads))
            out = P.Rows(ctx, np.full((pg.rows, heads, hd), 9.0), row_t)
            aq.paged_tree_attention(ctx, cache, b, dm.buf, words, heads, q.heads_struct(), out.heads_struct(), scale, window, None,
                                    ws)
            ctx.sync()
            assert np.all(np.abs(out.get() - want) <= limit)


@pytest.mark.parametrize("row_t,cache_t", PAIRS)
@pytest.mark.parametrize("new,window", [(6, 4), (70, 33)])
def test_chains_longer_than_the_window(ctx, row_t, cache_t, new, window):
    """A tree without branches: paged_attention's outputs up to the row that fills the window; the rows after it see their
    whole path and nothing before it."""
    print(f"long chain {row_t}/{cache_t} {new} window {window}", flush=True)
    rng = np.random.default_rng(window)
    heads, kv, hd = 4, 2, 128
    pg = P.Paged(ctx, rng, [new], [new + 100], kv, hd, 16, cache_t)
    masks = [np.arange(new) <= i for i in range(new)]
    q = P.Rows(ctx, rng.standard_normal((new, heads, hd)), row_t)
    scale, words = float(np.float32(1.0 / math.sqrt(hd))), -(-new // 32)
    want, parts = T.tree_attention(pg, masks, q.values(), scale, window)
    run, run_parts = P.attention(pg, q.values(), scale, window)
    limit, run_limit = (P.bound(x, y, row_t, cache_t, hd) for x, y in ((parts, want), (run_parts, run)))
    assert np.array_equal(parts[2], [max(window, i + 1) for i in range(new)])
    assert np.abs(want[window:] - run[window:]).max() > 0.1  # another row of values
    cache, batch = pg.structs()
    dm = P.Dev(ctx, T.pack(masks, words))
    ws = aq.DeviceBuffer(ctx, aq.paged_attention_workspace(ctx, cache, batch, heads))
    tree, chain = (P.Rows(ctx, np.full((new, heads, hd), 9.0), row_t) for _ in range(2))
    aq.paged_tree_attention(ctx, cache, batch, dm.buf, words, heads, q.heads_struct(), tree.heads_struct(), scale, window, None, ws)
    aq.paged_attention(ctx, cache, batch, heads, q.heads_struct(), chain.heads_struct(), scale, window, None, ws)
    ctx.sync()
    assert np.all(np.abs(tree.get() - want) <= limit) and np.all(np.abs(chain.get() - run) <= run_limit)
    assert np.all(np.abs(tree.get() - chain.get())[:window] <= (limit + run_limit)[:window])


@pytest.mark.parametrize("kv,hd", [(1, 8), (1, 64), (33, 8), (3, 168), (13, 40), (5, 104), (25, 64), (26, 80), (31, 128), (65, 64)])
def test_paths_over_rows_of_any_size(ctx, kv, hd):
    """1, 8, 33, 63, 65, 200, 260, 496 and 520 pieces of 16 bytes in a row: waves with lanes, and whole waves, that have none.
    Paths of more entries than a wave has lanes, and than are on their way together."""
    print(f"commit {kv} x {hd}", flush=True)
    rng = np.random.default_rng(kv * hd)
    new, keep = [100, 12, 3], [70, 9, 2]
    pg = P.Paged(ctx, rng, new, [130, 20, 40], kv, hd, 4, "bf16")
    paths = np.full((3, 80), -1, np.int32)
    for s in range(3):
        paths[s, : keep[s]] = np.sort(rng.choice(new[s], keep[s], replace=False))
    dp, dm = P.Dev(ctx, paths), P.Dev(ctx, np.array(keep, np.int32))
    cache, batch = pg.structs()
    aq.paged_tree_commit(ctx, cache, batch, dp.buf, dm.buf, 80)
    ctx.sync()
    k, v = pg.k.copy(), pg.v.copy()
    for s in range(3):
        base = pg.lens[s] - new[s]
        for i in range(keep[s]):
            a, to = pg.row_of(s, base + int(paths[s, i])), pg.row_of(s, base + i)
            k[to], v[to] = k[a], v[a]
    got = pg.pools()
    assert np.array_equal(got[0], k, equal_nan=True) and np.array_equal(got[1], v, equal_nan=True)


@pytest.mark.parametrize("in_place", [True, False])
def test_tables_of_arrays_side_by_side(ctx, in_place):
    """All arrays of the call in one allocation, each from where the one before ends: nothing lies over another."""
    print(f"side by side, in place {in_place}", flush=True)
    rng = np.random.default_rng(4)
    n, cols, pool, page, rows = 7, 5, 30, 4, 41
    w = T.Tables(n, cols, pool, page)
    w.ring = rng.permutation(pool).astype(np.int32)
    new = [6, 0, 9, 3, 12, 1, 7]
    sizes = {"slots": 2 * rows, "pages": n * cols, "held": n, "held_out": n, "ring": pool, "state": 4, "state_out": 4, "before": n,
             "new": n, "start": n + 1, "len": n, "missing": n, "pos": rows, "depth": rows}
    first = dict(zip(sizes, np.concatenate([[0], np.cumsum(list(sizes.values()))])))
    whole = np.zeros(sum(sizes.values()), np.int32)
    depth = rng.integers(0, 5, rows)
    for name, x in (("pages", w.pages.ravel()), ("ring", w.ring), ("state", [0, pool, 0, 0]), ("new", new), ("depth", depth)):
        whole[first[name]: first[name] + sizes[name]] = x
    d = P.Dev(ctx, whole)
    at = {name: d.buf.p.value + 4 * int(i) for name, i in first.items()}
    t = aq.page_tables(n, cols, pool, page, at["pages"], at["held"], at["ring"], at["state"], None if in_place else at["held_out"],
                       None if in_place else at["state_out"])
    length = "before" if in_place else "len"
    aq.paged_tables(ctx, t, at["before"], at["new"], rows, at["start"], at[length], at["missing"], at["pos"], at["slots"],
                    at["depth"])
    ctx.sync()
    got = d.get()
    want = dict(zip(("start", length, "missing", "pos", "slots"), w.step(np.zeros(n), new, rows, depth)))
    out = "" if in_place else "_out"
    want.update({"pages": w.pages, "ring": w.ring, "held" + out: w.held, "state" + out: [w.first, w.count, 0, 0], "new": new,
                 "depth": depth})
    for name, x in want.items():
        x = np.ascontiguousarray(x, np.int64).view(np.int32) if name == "slots" else np.ravel(x)
        assert np.array_equal(got[first[name]: first[name] + sizes[name]], x), name


@pytest.mark.parametrize("t", ["bf16", "f32"])
def test_more_work_groups_than_one_dimension_has(ctx, t):
    """More than 2^22 waves: a grid of two dimensions, whose last work-groups have no row. The rows repeat, at a distance that no
    power of two of rows is a multiple of, so a row taken for another shows."""
    rows, hd, again = (1 << 22) + 4099, 8, 1009
    print(f"norm {t} of {rows} rows", flush=True)
    rng = np.random.default_rng(11)
    x = rng.standard_normal((again, 1, hd))
    w = (1 + 0.3 * rng.standard_normal(hd)).astype(np.float32)
    few = P.Rows(ctx, x, t)
    stored, which = few.stored().reshape(again, hd), np.arange(rows) % again
    many, out = P.Dev(ctx, stored[which]), P.Dev(ctx, np.full((rows + 9, hd), 5, stored.dtype))
    dw = P.Dev(ctx, w)
    h = [aq.heads(d.buf, P.TYPES[t], hd, hd) for d in (many, out)]
    aq.qk_norm_rope(ctx, h[0], h[1], 1, None, None, 0, hd, rows, dw.buf, None, EPS)
    ctx.sync()
    got = out.get()
    want = T.normed(few.values(), w.astype(np.float64), EPS)
    limit = T.norm_bound(few.values(), w.astype(np.float64), EPS, want, t)
    assert np.all(np.abs(P.values(got[:again], t) - want[:, 0]) <= limit[:, 0])
    assert np.array_equal(got[:rows], got[:again][which]) and np.all(got[rows:] == 5)


@pytest.mark.parametrize("cache_t", ["f16", "f32"])
def test_a_pool_that_runs_out(ctx, cache_t):
    """Requests that want more pages than there are, step by step: paths end before the first row without a slot, so that every
    position that counts was stored, and requests that waited go on when another's pages come back."""
    print(f"short pool {cache_t}", flush=True)
    rng = np.random.default_rng(6)
    n, cols, pool, page, kv, hd, most, goal = 4, 8, 13, 4, 1, 16, 6, [20, 24, 14, 17]
    rows = n * most
    dev = lambda a: P.Dev(ctx, a)  # noqa: E731
    pages, held, ring = dev(np.full((n, cols), -1, np.int32)), dev(np.zeros(n, np.int32)), dev(np.arange(pool, dtype=np.int32))
    state, before, new, start = (dev(x) for x in (np.array([0, pool, 0, 0], np.int32), np.zeros(n, np.int32), np.zeros(n, np.int32),
                                                  np.zeros(n + 1, np.int32)))
    length, missing, pos, slots = (dev(np.zeros(*x)) for x in ((n, np.int32), (n, np.int32), (rows, np.int32), (rows, np.int64)))
    nan = P.store(np.full((pool, page, kv, hd), np.nan), cache_t)
    k, v = dev(nan), dev(nan)
    cache = aq.paged_kv(k.buf, v.buf, P.TYPES[cache_t], pool, page, kv, hd)
    batch = aq.paged_batch(n, start.buf, length.buf, pages.buf, cols, rows, most, cols * page)
    t = aq.page_tables(n, cols, pool, page, pages.buf, held.buf, ring.buf, state.buf)
    lens, done, waited, went_on = np.zeros(n, np.int64), np.zeros(n, bool), np.zeros(n, bool), np.zeros(n, bool)
    for step in range(60):
        count = np.where(done, -1, np.minimum(rng.integers(2, most + 1, n), cols * page - lens))
        new.buf.upload(count.astype(np.int32))
        aq.paged_tables(ctx, t, before.buf, new.buf, rows, start.buf, length.buf, missing.buf, pos.buf, slots.buf)
        ctx.sync()
        first, slot, short = start.get(), slots.get(), missing.get()
        # the tree's row j is accepted for the j-th of some rising choice; the stored value says whose and which position
        path, m = np.full((n, most), -1, np.int32), np.zeros(n, np.int32)
        x = np.full((rows, kv, hd), 99.0)
        for s in range(n):
            c = max(int(count[s]), 0)
            take = np.sort(rng.choice(c, rng.integers(1, c + 1), replace=False)) if c else np.zeros(0, int)
            for i, j in enumerate(take):
                x[first[s] + j] = s * 64 + lens[s] + i
            fits = [j for j in take if slot[first[s] + j] >= 0]
            path[s, : len(fits)], m[s] = fits, len(fits)
            went_on[s] |= waited[s] and len(fits) > 0
            waited[s] |= len(fits) < len(take)
            assert (short[s] > 0) >= (len(fits) < len(take))
        r, dp, dm = P.Rows(ctx, x, cache_t), dev(path), dev(m)
        aq.paged_append(ctx, cache, batch, r.heads_struct(), r.heads_struct())
        aq.paged_tree_commit(ctx, cache, batch, dp.buf, dm.buf, most, before.buf)
        ctx.sync()
        lens = np.where(done, 0, lens + m)
        assert before.get().tolist() == lens.tolist()
        table, got = pages.get(), [P.values(p.get().reshape(pool, page, kv, hd), cache_t) for p in (k, v)]
        for s in range(n):
            for p in range(int(lens[s])):
                assert all(np.all(g[table[s, p // page], p % page] == s * 64 + p) for g in got), (step, s, p)
        done |= lens >= goal
        if done.all():
            break
    assert done.all() and went_on.any()
