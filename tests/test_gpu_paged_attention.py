"""Attention over a paged cache on the device against its definition in 64 bits: every pair of row and cache types, head
shapes and sizes (odd ones among them), one token to several row tiles, pages that end inside a tile, windows, gates,
strides, holes, rows that see nothing, and infinities and NaN wherever a row does not look. Tolerances: paged_plain.bound,
by arithmetic from the roundings of each step."""
import ctypes as C
import math

import numpy as np
import pytest

import aqueduct as aq
import paged_plain as P

pytestmark = pytest.mark.gpu
PAIRS = [("f32", "f32"), ("f32", "f16"), ("f32", "bf16"), ("f16", "f16"), ("bf16", "bf16")]


@pytest.fixture(scope="module")
def ctx():
    return aq.Context(0)


ENOUGH = 5 << 20  # rows x heads x positions past which many 16-bit rows go to a kernel of their own
SHORT = 512       # positions up to which a work-group may have whole sequences


def bounds(pg, q):
    """The batch's bounds as they are and, where that changes the kernel or the division of the work, with wide tables and
    a large max_len."""
    reach = min(pg.max_len, pg.cols * pg.page)
    many = q.t != "f32" and pg.max_rows * (q.heads // pg.kv) > 32 and pg.rows * q.heads * reach <= ENOUGH
    return (False, True) if many or reach <= SHORT else (False,)


def run(ctx, pg, q, out, scale, window=0, gate=None, stream=None, sync=True, loose=False):
    cache, batch = pg.structs()
    if loose:
        positions = max(ENOUGH // (pg.rows * q.heads) + 1, 4 * SHORT)
        wide = P.Dev(ctx, np.full((len(pg.lens), max(pg.cols, -(-positions // pg.page))), 10 ** 9, np.int32))
        wide.buf.upload(np.concatenate([pg.table, wide.get()[:, pg.cols:]], 1))
        batch = aq.paged_batch(len(pg.lens), pg.dstarts.buf, pg.dlens.buf, wide.buf, wide.shape[1], pg.rows, pg.max_rows,
                               max(positions, pg.max_len))
    ws = aq.DeviceBuffer(ctx, aq.paged_attention_workspace(ctx, cache, batch, q.heads))
    aq.paged_attention(ctx, cache, batch, q.heads, q.heads_struct(), out.heads_struct(), scale, window,
                       gate.heads_struct() if gate else None, ws, stream=stream)
    if sync:
        ctx.sync()
    return ws


def check(ctx, seed, new, lens, heads, kv, hd, page, row_t, cache_t, window=0, gated=False, pad=0, skip=0, qs=1.5, **kw):
    print(f"attention {row_t}/{cache_t} new {new} lens {lens} heads {heads}/{kv} x {hd} page {page} window {window} "
          f"gate {gated} pad {pad} skip {skip} {kw}", flush=True)
    rng = np.random.default_rng(seed)
    pg = P.Paged(ctx, rng, new, lens, kv, hd, page, cache_t, **kw)
    q = P.Rows(ctx, rng.standard_normal((pg.rows, heads, hd)) * qs, row_t, pad, skip)
    gate = P.Rows(ctx, rng.standard_normal((pg.rows, heads, hd)) * 2, row_t, pad, skip) if gated else None
    scale = float(np.float32(1.0 / math.sqrt(hd)))
    want, parts = P.attention(pg, q.values(), scale, window, gate.values() if gated else None)
    for loose in bounds(pg, q):
        out = P.Rows(ctx, np.full((pg.rows, heads, hd), 9.0), row_t, pad, skip)
        run(ctx, pg, q, out, scale, window, gate, loose=loose)
        compare(pg, out.get(), want, P.bound(parts, want, row_t, cache_t, hd))


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
def test_single_tokens(ctx, row_t, cache_t, heads, kv, hd):
    check(ctx, heads + hd, [1, 1, 1], [1, 130, 777], heads, kv, hd, 16, row_t, cache_t)


@pytest.mark.parametrize("row_t,cache_t", PAIRS)
@pytest.mark.parametrize("heads,kv,hd,new", [(4, 2, 64, 4), (8, 2, 128, 3), (24, 4, 256, 4), (4, 4, 96, 7), (4, 1, 256, 8)])
def test_verify_batches(ctx, row_t, cache_t, heads, kv, hd, new):
    check(ctx, heads * new, [new, 1, new], [new, 64, 301], heads, kv, hd, 24, row_t, cache_t)


@pytest.mark.parametrize("row_t,cache_t", PAIRS)
@pytest.mark.parametrize("heads,kv,hd,new", [(4, 2, 64, 70), (8, 2, 128, 65), (6, 1, 256, 40), (5, 5, 72, 130), (3, 1, 160, 33)])
def test_prompt_chunks(ctx, row_t, cache_t, heads, kv, hd, new):
    check(ctx, heads * new, [new, 2, new + 9], [new, 150, 400], heads, kv, hd, 16, row_t, cache_t)


@pytest.mark.parametrize("row_t,cache_t", PAIRS)
@pytest.mark.parametrize("window", [1, 5, 32, 129, 100000])
@pytest.mark.parametrize("new", [1, 5, 90])
def test_windows(ctx, row_t, cache_t, window, new):
    check(ctx, window + new, [new, new], [new + 3, 500], 4, 2, 128, 16, row_t, cache_t, window=window)


@pytest.mark.parametrize("page", [1, 7, 16, 32, 100, 1024])
@pytest.mark.parametrize("row_t,cache_t", [("bf16", "bf16"), ("f32", "f32")])
@pytest.mark.parametrize("new", [1, 50])
def test_page_sizes_and_layouts(ctx, page, row_t, cache_t, new):
    check(ctx, page, [new, new], [333, new], 4, 2, 64, page, row_t, cache_t, layout="heads")
    check(ctx, page, [new, new], [333, new], 4, 2, 64, page, row_t, cache_t, extra=0)


@pytest.mark.parametrize("row_t,cache_t", PAIRS)
@pytest.mark.parametrize("new", [1, 4, 60])
@pytest.mark.parametrize("pad,skip", [(0, 0), (64, 0), (1, 3)])
def test_gates_and_strides(ctx, row_t, cache_t, new, pad, skip):
    check(ctx, pad + new, [new], [200], 6, 2, 128, 16, row_t, cache_t, gated=True, pad=pad, skip=skip)


@pytest.mark.parametrize("row_t,cache_t", PAIRS)
@pytest.mark.parametrize("most", [1, 40])
def test_empty_sequences_and_rows_that_see_nothing(ctx, row_t, cache_t, most):
    """Sequences without rows, of length 0, with more rows than positions; rows behind the last sequence."""
    new = [0, 1, 0, min(3, most), most, 0]
    lens = [50, 0, 0, 1, most, 9]
    check(ctx, 3, new, lens, 4, 2, 64, 16, row_t, cache_t, n_rows=sum(new) + 3)


@pytest.mark.parametrize("row_t,cache_t", PAIRS)
@pytest.mark.parametrize("new", [1, 3, 40])
def test_holes(ctx, row_t, cache_t, new):
    """Table entries outside the pool, positions past the table and past max_len are not attended; a row of holes is 0."""
    rng = np.random.default_rng(5)
    pg = P.Paged(ctx, rng, [new, new, new], [300, 100, 64], 2, 64, 16, cache_t)
    pg.table[0, 3] = -1
    pg.table[0, 5] = pg.k.shape[0]
    pg.table[0, 7] = 2 ** 31 - 1
    pg.table[0, 17:] = -7
    pg.table[2, :] = -1
    pg.upload()
    x = np.zeros((20000, 4, 64))
    x[: pg.rows] = rng.standard_normal((pg.rows, 4, 64))
    shapes = [(cols, max_len, n_rows) for n_rows in (pg.rows, 20000) for cols, max_len in
              ((pg.cols, 300), (5, 300), (pg.cols, 90))]
    for cols, max_len, n_rows in shapes[: 6 if new == 40 and row_t != "f32" else 3]:
        print(f"holes {row_t}/{cache_t} new {new} cols {cols} max_len {max_len} of {n_rows} rows", flush=True)
        short = P.Paged.__new__(P.Paged)
        short.__dict__.update(pg.__dict__, cols=cols, max_len=max_len, rows=n_rows,
                              table=np.ascontiguousarray(pg.table[:, :cols]))
        short.dtable = P.Dev(ctx, short.table)
        q, out = P.Rows(ctx, x[:n_rows], row_t), P.Rows(ctx, np.full((n_rows, 4, 64), 9.0), row_t)
        run(ctx, short, q, out, 0.125)
        want, parts = P.attention(short, q.values(), 0.125)
        compare(short, out.get(), want, P.bound(parts, want, row_t, cache_t, 64))
        assert np.all(out.get()[2 * new: 3 * new] == 0.0)


@pytest.mark.parametrize("row_t,cache_t", PAIRS)
@pytest.mark.parametrize("new,window", [(1, 0), (1, 6), (4, 0), (4, 6), (60, 0), (60, 40)])
@pytest.mark.parametrize("bad", [np.inf, -np.inf, np.nan])
def test_what_a_row_does_not_see_never_reaches_it(ctx, row_t, cache_t, new, window, bad):
    """Values and keys that are not finite, at positions that only some rows of a tile see: the others are as without
    them; the rows that see an infinite value get it."""
    print(f"odd values {row_t}/{cache_t} new {new} window {window} {bad}", flush=True)
    rng = np.random.default_rng(11)
    pg = P.Paged(ctx, rng, [new], [150], 2, 128, 16, cache_t)
    at = [150 - 1, 150 - new // 2, 150 - new - 3]  # the last row's alone; half the rows'; all (or the window's)
    if new == 1:
        at = [150 - 1, 150, 150 - 8]  # its own; past it; all positions but the window's
    for i, p in enumerate(at):
        pg.v[pg.row_of(0, p)][i % 2, 5 + 40 * i] = bad
    if window:
        pg.k[pg.row_of(0, 150 - new - window)] = bad  # before all windows
    pg.upload()
    q = P.Rows(ctx, rng.standard_normal((new, 4, 128)), row_t)
    want, parts = P.attention(pg, q.values(), 0.08, window)
    limit = P.bound(tuple(np.nan_to_num(x, posinf=0, neginf=0) for x in parts), np.nan_to_num(want, posinf=0, neginf=0),
                    row_t, cache_t, 128)
    fine = np.isfinite(want)
    for loose in bounds(pg, q):
        out = P.Rows(ctx, np.full((new, 4, 128), 9.0), row_t)
        run(ctx, pg, q, out, 0.08, window, loose=loose)
        got = out.get()
        assert np.array_equal(fine, np.isfinite(got))
        assert np.array_equal(np.isnan(want), np.isnan(got)) and np.array_equal(want[~fine & ~np.isnan(want)],
                                                                                got[~fine & ~np.isnan(want)])
        assert np.all(np.abs(got[fine] - want[fine]) <= limit[fine])
    pg.v = np.where(np.isfinite(pg.v), pg.v, 0.5)
    pg.k[pg.row_of(0, 149)] = bad  # a key that only the last row sees
    pg.upload()
    pg.k = np.where(np.isfinite(pg.k), pg.k, 0.0)  # for the definition; the device keeps the others
    want, parts = P.attention(pg, q.values(), 0.08, window)
    for loose in bounds(pg, q):
        out = P.Rows(ctx, np.full((new, 4, 128), 9.0), row_t)
        run(ctx, pg, q, out, 0.08, window, loose=loose)
        got = out.get()
        assert np.all(np.isfinite(got[:-1]))
        assert np.all(np.abs(got - want)[:-1] <= P.bound(parts, want, row_t, cache_t, 128)[:-1])


@pytest.mark.parametrize("row_t,cache_t", PAIRS)
@pytest.mark.parametrize("new", [1, 40])
def test_infinite_keys(ctx, row_t, cache_t, new):
    """A key with an infinite value scores plus or minus infinity: a NaN row, or one that leaves the position out."""
    rng = np.random.default_rng(12)
    pg = P.Paged(ctx, rng, [new], [150], 2, 128, 16, cache_t)
    pg.k[pg.row_of(0, 70)][:, 9] = np.inf
    pg.upload()
    q = P.Rows(ctx, rng.standard_normal((new, 4, 128)), row_t)
    up, gots = q.values()[..., 9] > 0, []
    for loose in bounds(pg, q):
        out = P.Rows(ctx, np.full((new, 4, 128), 9.0), row_t)
        run(ctx, pg, q, out, 0.08, loose=loose)
        gots.append(out.get())
        assert np.array_equal(np.isnan(gots[-1]).all(-1), up) and np.array_equal(np.isnan(gots[-1]).any(-1), up)
    pg.v[pg.row_of(0, 70)] = 0
    pg.k[pg.row_of(0, 70)] = 0
    want, parts = P.attention(pg, q.values(), 0.08)
    # position 70 has score 0 and value 0 there: its weight is taken out of the sum
    weight = np.zeros(want.shape[:2])
    for r in range(new):
        pos = 150 - new + r
        places = np.array([pg.row_of(0, p) for p in range(pos + 1)])
        for h in range(4):
            x = pg.k[places[:, 0], places[:, 1], h // 2] @ q.values()[r, h] * 0.08
            weight[r, h] = 1.0 / np.exp(x).sum() if pos >= 70 else 0.0
    want = want / (1 - weight[..., None])
    parts = (parts[0] / (1 - weight[..., None]), *parts[1:])
    for got in gots:
        assert np.all((np.abs(got - want) <= P.bound(parts, want, row_t, cache_t, 128))[~up])


@pytest.mark.parametrize("row_t,cache_t", PAIRS)
@pytest.mark.parametrize("qs,sigma", [(1e-6, 1.0), (40.0, 1.0), (300.0, 100.0), (1.0, 1e-3)])
@pytest.mark.parametrize("new", [1, 50])
def test_score_ranges(ctx, row_t, cache_t, qs, sigma, new):
    """Flat and one-hot softmaxes; queries past f16's range over an f16 cache."""
    if row_t == "f32" and qs == 300.0:
        qs = 1e6
    check(ctx, 21, [new], [260], 4, 2, 128, 16, row_t, cache_t, qs=qs, sigma=sigma)


@pytest.mark.parametrize("row_t,cache_t", PAIRS)
def test_long_context_split_over_the_chip(ctx, row_t, cache_t):
    check(ctx, 31, [1, 1], [9001, 5], 6, 1, 128, 32, row_t, cache_t)
    check(ctx, 31, [20, 1], [5003, 2500], 4, 1, 64, 64, row_t, cache_t, window=3000)


@pytest.mark.parametrize("row_t,cache_t", [("bf16", "bf16"), ("f32", "f16")])
@pytest.mark.parametrize("n", [1100, 2049])
def test_many_sequences(ctx, row_t, cache_t, n):
    """More sequences than one work-group divides by itself."""
    rng = np.random.default_rng(2)
    lens = [int(x) for x in rng.integers(1, 9, n)]
    lens[n // 2] = 300
    check(ctx, 1, [1] * n, lens, 2, 1, 64, 8, row_t, cache_t)


@pytest.mark.parametrize("row_t,cache_t", PAIRS)
def test_the_same_call_gives_the_same_bits(ctx, row_t, cache_t):
    rng = np.random.default_rng(8)
    for new in ([1, 1, 1], [50, 3, 9]):
        pg = P.Paged(ctx, rng, new, [1500, 40, 700], 2, 128, 16, cache_t)
        q = P.Rows(ctx, rng.standard_normal((pg.rows, 8, 128)), row_t)
        for loose in bounds(pg, q):
            got = []
            for _ in range(3):
                out = P.Rows(ctx, np.full((pg.rows, 8, 128), 9.0), row_t)
                run(ctx, pg, q, out, 0.09, loose=loose)
                got.append(out.dev.get())
            assert all(np.array_equal(got[0].view(np.uint8), x.view(np.uint8)) for x in got[1:])


@pytest.mark.parametrize("row_t,cache_t", PAIRS)
def test_in_place(ctx, row_t, cache_t):
    """The output over the queries, and over the gate."""
    rng = np.random.default_rng(9)
    for new in ([1, 1], [40, 3]):
        pg = P.Paged(ctx, rng, new, [700, 90], 2, 64, 16, cache_t)
        x, gx = rng.standard_normal((2, pg.rows, 4, 64))
        q, gate = P.Rows(ctx, x, row_t), P.Rows(ctx, gx, row_t)
        want, parts = P.attention(pg, q.values(), 0.125, 0, gate.values())
        for over, loose in [(o, b) for o in ("q", "gate") for b in bounds(pg, q)]:
            q, gate = P.Rows(ctx, x, row_t), P.Rows(ctx, gx, row_t)
            out = q if over == "q" else gate
            run(ctx, pg, q, out, 0.125, 0, gate, loose=loose)
            assert np.all(np.abs(out.get() - want) <= P.bound(parts, want, row_t, cache_t, 64)), over
