"""Attention of trees over a paged cache on the device against its definition in 64 bits: every pair of row and cache types,
head shapes, trees of one row to several row tiles and mask words, contexts that end anywhere in a tile, windows, gates,
strides, holes, masks that leave a row nothing, and infinities and NaN wherever a row does not look. Tolerances:
paged_plain.bound, by arithmetic from the roundings of each step."""
import math

import numpy as np
import pytest

import aqueduct as aq
import paged_plain as P
import tree_plain as T

pytestmark = pytest.mark.gpu
PAIRS = [("f32", "f32"), ("f32", "f16"), ("f32", "bf16"), ("f16", "f16"), ("bf16", "bf16")]
ENOUGH = 5 << 20  # rows x heads x positions past which many 16-bit rows go to a kernel of their own
SHORT = 512       # positions up to which a work-group may have whole sequences


@pytest.fixture(scope="module")
def ctx():
    return aq.Context(0)


def attend(ctx, pg, masks, words, q, out, scale, window=0, gate=None, loose=False):
    """One call; `loose`: with wide tables and a large max_len, which change the kernel or the division of the work."""
    cache, batch = pg.structs()
    if loose:
        positions = max(ENOUGH // (pg.rows * q.heads) + 1, 4 * SHORT)
        table = np.full((len(pg.lens), max(pg.cols, -(-positions // pg.page))), 10 ** 9, np.int32)
        table[:, : pg.cols] = pg.table
        wide = P.Dev(ctx, table)
        batch = aq.paged_batch(len(pg.lens), pg.dstarts.buf, pg.dlens.buf, wide.buf, wide.shape[1], pg.rows, pg.max_rows,
                               max(positions, pg.max_len))
    ws = aq.DeviceBuffer(ctx, aq.paged_attention_workspace(ctx, cache, batch, q.heads))
    ws.upload(np.full(ws.nbytes, 0xFF, np.uint8))
    dm = P.Dev(ctx, T.pack(masks, words))
    aq.paged_tree_attention(ctx, cache, batch, dm.buf, words, q.heads, q.heads_struct(), out.heads_struct(), scale, window,
                            gate.heads_struct() if gate else None, ws)
    ctx.sync()


def check(ctx, seed, new, lens, heads, kv, hd, page, row_t, cache_t, window=0, gated=False, pad=0, skip=0, qs=1.5, masks=None,
          words=0, **kw):
    print(f"tree {row_t}/{cache_t} new {new} lens {lens} heads {heads}/{kv} x {hd} page {page} window {window} gate {gated} "
          f"pad {pad} skip {skip} words {words} {kw}", flush=True)
    rng = np.random.default_rng(seed)
    pg = P.Paged(ctx, rng, new, lens, kv, hd, page, cache_t, **kw)
    masks = T.random_trees(rng, new) if masks is None else masks(rng)
    masks = masks + [np.ones(1, bool)] * (pg.rows - len(masks))
    words = words or -(-max(pg.max_rows, 1) // 32)
    q = P.Rows(ctx, rng.standard_normal((pg.rows, heads, hd)) * qs, row_t, pad, skip)
    gate = P.Rows(ctx, rng.standard_normal((pg.rows, heads, hd)) * 2, row_t, pad, skip) if gated else None
    scale = float(np.float32(1.0 / math.sqrt(hd)))
    want, parts = T.tree_attention(pg, masks, q.values(), scale, window, gate.values() if gated else None)
    limit = P.bound(parts, want, row_t, cache_t, hd)
    outs = []
    for loose in (False, True):
        out = P.Rows(ctx, np.full((pg.rows, heads, hd), 9.0), row_t, pad, skip)
        attend(ctx, pg, masks, words, q, out, scale, window, gate, loose)
        outs.append(out.get())
        compare(pg, outs[-1], want, limit)
    return pg, masks, q, want, limit, outs


def compare(pg, got, want, bound):
    used = min(int(pg.starts[-1]), pg.rows)
    assert np.all(got[used:] == 9.0), "rows behind the last sequence"
    got, want, bound = got[:used], want[:used], bound[:used]
    assert np.all(np.isfinite(got)), f"{np.sum(~np.isfinite(got))} of {got.size} not finite"
    off = np.abs(got - want)
    worst = np.unravel_index(np.argmax(off - bound), off.shape) if off.size else None
    assert np.all(off <= bound), f"at {worst}: {got[worst]} for {want[worst]}, off {off[worst]:.3g} over {bound[worst]:.3g}"


@pytest.mark.parametrize("row_t,cache_t", PAIRS)
@pytest.mark.parametrize("heads,kv,hd", [(4, 2, 64), (6, 1, 128), (24, 4, 256), (5, 5, 80), (3, 1, 8), (40, 2, 192)])
@pytest.mark.parametrize("new", [1, 5, 27])
def test_trees(ctx, row_t, cache_t, heads, kv, hd, new):
    check(ctx, heads + hd + new, [new, new, 1, new], [new, 130, 777, 300 + new], heads, kv, hd, 16, row_t, cache_t)


@pytest.mark.parametrize("row_t,cache_t", PAIRS)
@pytest.mark.parametrize("heads,kv,hd", [(4, 2, 64), (8, 2, 128), (6, 1, 256)])
@pytest.mark.parametrize("new", [33, 64, 130, 257])
def test_large_trees(ctx, row_t, cache_t, heads, kv, hd, new):
    check(ctx, hd * new, [new, 2, new - 9], [new + 95, 150, 400], heads, kv, hd, 16, row_t, cache_t)


@pytest.mark.parametrize("row_t,cache_t", PAIRS)
@pytest.mark.parametrize("before", list(range(0, 36, 5)) + [63, 64, 65, 127, 128, 129])
def test_where_the_context_ends(ctx, row_t, cache_t, before):
    """Every offset of the tree inside a tile of 16, 32 or 64 positions."""
    check(ctx, before, [20, 40], [before + 20, before + 41], 4, 2, 128, 16, row_t, cache_t)
    check(ctx, before, [20, 40], [before + 20, before + 41], 4, 2, 256, 8, row_t, cache_t)


@pytest.mark.parametrize("row_t,cache_t", PAIRS)
@pytest.mark.parametrize("window", [1, 3, 32, 129, 100000])
@pytest.mark.parametrize("new", [6, 90])
def test_windows(ctx, row_t, cache_t, window, new):
    check(ctx, window + new, [new, new], [new + 3, 500], 4, 2, 128, 16, row_t, cache_t, window=window)


@pytest.mark.parametrize("row_t,cache_t", PAIRS)
@pytest.mark.parametrize("new", [5, 40])
def test_gates_and_strides(ctx, row_t, cache_t, new):
    for pad, skip in ((0, 0), (8, 0), (1, 3)):
        check(ctx, new, [new, 3], [200, 90], 8, 2, 128, 16, row_t, cache_t, gated=True, pad=pad, skip=skip,
              layout="heads" if pad else "slots", n_rows=new + 5)


@pytest.mark.parametrize("row_t,cache_t", PAIRS)
@pytest.mark.parametrize("new", [4, 70])
def test_any_mask(ctx, row_t, cache_t, new):
    """Masks of no tree: none of a row's bits, all of them, any, later rows, rows that do not see themselves, more words
    than the rows need; over nothing before them, where a row with no bit sees nothing, and over something."""
    def masks(rng):
        rows = []
        for n in (new, new, 2):
            m = rng.random((n, n)) < 0.4
            m[0], m[n - 1], m[n // 2] = False, True, False
            rows += list(m)
        return rows
    check(ctx, new, [new, new, 2], [new, 100 + new, 2], 4, 2, 64, 16, row_t, cache_t, masks=masks, words=5)
    check(ctx, new, [new, new, 2], [new, 100 + new, 2], 4, 2, 256, 16, row_t, cache_t, masks=masks, words=3, window=50)


@pytest.mark.parametrize("row_t,cache_t", PAIRS)
@pytest.mark.parametrize("new", [6, 70])
def test_chains_are_paged_attention(ctx, row_t, cache_t, new):
    """A tree without branches: what aq_paged_attention gives, within the bound of both."""
    def chain(rng):
        return [np.arange(n) <= i for n in (new, 3) for i in range(n)]
    pg, _, q, want, limit, outs = check(ctx, new, [new, 3], [new + 200, 77], 8, 2, 128, 16, row_t, cache_t, masks=chain)
    cache, batch = pg.structs()
    out = P.Rows(ctx, np.full((pg.rows, 8, 128), 9.0), row_t)
    ws = aq.DeviceBuffer(ctx, aq.paged_attention_workspace(ctx, cache, batch, 8))
    aq.paged_attention(ctx, cache, batch, 8, q.heads_struct(), out.heads_struct(), float(np.float32(1 / math.sqrt(128))), 0,
                       None, ws)
    ctx.sync()
    assert np.all(np.abs(out.get() - outs[0]) <= 2 * limit)


@pytest.mark.parametrize("row_t,cache_t", PAIRS)
@pytest.mark.parametrize("heads,kv,hd", [(4, 2, 64), (4, 2, 128), (4, 1, 256), (5, 5, 80)])
@pytest.mark.parametrize("new", [7, 70])
def test_what_is_hidden_never_reaches_a_row(ctx, row_t, cache_t, heads, kv, hd, new):
    """Infinities, NaN and the type's lowest and largest values in the K and V of rows that a mask hides, of positions that
    the window leaves out, and of pages nobody has."""
    print(f"hidden {row_t}/{cache_t} {heads}/{kv} x {hd} new {new}", flush=True)
    rng = np.random.default_rng(hd + new)
    big = {"f32": 3e38, "f16": 65504.0, "bf16": 3e38}[cache_t]
    odd = np.array([np.inf, -np.inf, np.nan, -big, big])
    for window in (0, 40):
        pg = P.Paged(ctx, rng, [new, new], [new + 90, new + 7], kv, hd, 16, cache_t)
        masks = T.random_trees(rng, pg.new)
        blind = [2, 5, new - 1]  # of each sequence: rows that only they themselves see, and they see no other odd one
        for s in range(2):
            for i in range(new):
                for b in blind:
                    masks[int(pg.starts[s]) + i][b] = False
        for s in range(2):
            base = pg.lens[s] - new
            for j, b in enumerate(blind):
                at = pg.row_of(s, base + b)
                pg.k[at][..., rng.integers(0, hd, 3)] = odd[(j + s) % 5]
                pg.v[at][..., rng.integers(0, hd, 3)] = odd[(j + 2 * s + 1) % 5]
            if window:  # no row of at most `new` bits sees these
                for p in range(max(0, base - window)):
                    pg.v[pg.row_of(s, p)][..., p % hd] = odd[p % 5]
                    pg.k[pg.row_of(s, p)][..., p % hd] = odd[(p + 1) % 5]
        pg.upload()
        q = P.Rows(ctx, rng.standard_normal((pg.rows, heads, hd)), row_t)
        scale = float(np.float32(1.0 / math.sqrt(hd)))
        want, parts = T.tree_attention(pg, masks, q.values(), scale, window)
        assert np.all(np.isfinite(want))
        limit = P.bound(parts, want, row_t, cache_t, hd)
        for loose in (False, True):
            out = P.Rows(ctx, np.full((pg.rows, heads, hd), 9.0), row_t)
            attend(ctx, pg, masks, -(-new // 32), q, out, scale, window, None, loose)
            compare(pg, out.get(), want, limit)


@pytest.mark.parametrize("row_t,cache_t", PAIRS)
@pytest.mark.parametrize("new", [7, 70])
def test_infinite_values_reach_those_that_see_them(ctx, row_t, cache_t, new):
    """An infinite value of a draft: infinite in the rows that see it, finite in the others."""
    rng = np.random.default_rng(new)
    pg = P.Paged(ctx, rng, [new, new], [new + 50, new], 2, 128, 16, cache_t)
    masks = T.random_trees(rng, pg.new)
    for s in range(2):
        pg.v[pg.row_of(s, pg.lens[s] - new + 3)][0, 5] = np.inf
    pg.upload()
    q = P.Rows(ctx, rng.standard_normal((pg.rows, 4, 128)), row_t)
    for loose in (False, True):
        out = P.Rows(ctx, np.full((pg.rows, 4, 128), 9.0), row_t)
        attend(ctx, pg, masks, -(-new // 32), q, out, 0.0884, 0, None, loose)
        got = out.get()
        sees = np.array([bool(m[3]) for m in masks])
        assert sees.any() and not sees.all()
        assert np.all(np.isposinf(got[sees][:, :2, 5])) and np.all(np.isfinite(got[~sees]))
        assert np.all(np.isfinite(np.delete(got, 5, -1))) and np.all(np.isfinite(got[:, 2:]))


@pytest.mark.parametrize("row_t,cache_t", PAIRS)
@pytest.mark.parametrize("new", [7, 70])
def test_holes(ctx, row_t, cache_t, new):
    """Pages that are not there, before the tree and inside it; lengths shorter than the new rows, zero and negative;
    positions past max_len."""
    print(f"holes {row_t}/{cache_t} new {new}", flush=True)
    rng = np.random.default_rng(new)
    lens = [new + 90, new - 3, 0, -5, new + 40]
    pg = P.Paged(ctx, rng, [new] * 5, lens, 2, 64, 4, cache_t, cols=-(-(new + 90) // 4), max_len=new + 60)
    pg.table[0, 3], pg.table[0, 4], pg.table[0, -3], pg.table[4, 2] = -1, 10 ** 9, -2 ** 31, pg.k.shape[0]
    pg.upload()
    masks = T.random_trees(rng, pg.new)
    q = P.Rows(ctx, rng.standard_normal((pg.rows, 4, 64)), row_t)
    want, parts = T.tree_attention(pg, masks, q.values(), 0.125)
    limit = P.bound(parts, want, row_t, cache_t, 64)
    out = P.Rows(ctx, np.full((pg.rows, 4, 64), 9.0), row_t)
    attend(ctx, pg, masks, -(-new // 32), q, out, 0.125)
    compare(pg, out.get(), want, limit)


@pytest.mark.parametrize("row_t,cache_t", PAIRS)
@pytest.mark.parametrize("new", [6, 40])
def test_rows_past_the_bounds_stay(ctx, row_t, cache_t, new):
    """A last sequence that the row tensors cut: its rows within them are right (they may see the keys of those behind), and
    nothing behind is written."""
    rng = np.random.default_rng(7)
    pg = P.Paged(ctx, rng, [new, new, new], [300, 200, 100], 2, 64, 16, cache_t)
    x = rng.standard_normal((pg.rows, 4, 64))
    q, out = P.Rows(ctx, x, row_t), P.Rows(ctx, np.full((pg.rows, 4, 64), 9.0), row_t)
    masks = [m | (rng.random(len(m)) < 0.3) for m in T.random_trees(rng, pg.new)]
    want, parts = T.tree_attention(pg, masks, q.values(), 0.125)
    limit = P.bound(parts, want, row_t, cache_t, 64)
    cache, _ = pg.structs()
    n = 2 * new + new // 2
    b = aq.paged_batch(3, pg.dstarts.buf, pg.dlens.buf, pg.dtable.buf, pg.cols, n, new, 300)
    ws = aq.DeviceBuffer(ctx, aq.paged_attention_workspace(ctx, cache, b, 4))
    words = -(-new // 32)
    dm = P.Dev(ctx, T.pack(masks[:n], words))
    aq.paged_tree_attention(ctx, cache, b, dm.buf, words, 4, q.heads_struct(), out.heads_struct(), 0.125, 0, None, ws)
    ctx.sync()
    got = out.get()
    assert np.all(got[n:] == 9.0) and np.all(np.abs(got - want)[:n] <= limit[:n])


@pytest.mark.parametrize("row_t,cache_t,n_seq,new", [("f32", "bf16", 350, 26), ("bf16", "bf16", 350, 26),
                                                     ("bf16", "bf16", 1100, 9)])
def test_more_row_tiles_than_one_work_group_divides(ctx, row_t, cache_t, n_seq, new):
    """The plan's own launch, few positions each."""
    rng = np.random.default_rng(6)
    lens = [int(n) for n in new + rng.integers(0, 9, n_seq)]
    check(ctx, 6, [new] * n_seq, lens, 4, 1, 16, 16, row_t, cache_t)


@pytest.mark.parametrize("row_t,cache_t", PAIRS)
def test_outputs_over_their_inputs(ctx, row_t, cache_t):
    """out over q, and over the gate: the bits of an output of its own."""
    rng = np.random.default_rng(3)
    pg = P.Paged(ctx, rng, [9, 12], [300, 40], 2, 64, 16, cache_t)
    masks = T.random_trees(rng, pg.new)
    x, g = (rng.standard_normal((pg.rows, 8, 64)) for _ in range(2))
    q, gate, out = P.Rows(ctx, x, row_t), P.Rows(ctx, g, row_t), P.Rows(ctx, np.zeros(x.shape), row_t)
    attend(ctx, pg, masks, 1, q, out, 0.125, 0, gate)
    attend(ctx, pg, masks, 1, q, q, 0.125, 0, gate)
    assert np.array_equal(q.get(), out.get())
    q = P.Rows(ctx, x, row_t)
    attend(ctx, pg, masks, 1, q, gate, 0.125, 0, gate)
    assert np.array_equal(gate.get(), out.get())
