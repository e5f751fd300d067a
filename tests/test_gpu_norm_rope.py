"""The heads' norms with the rotation on the device, over rows and into pages, against their formulas in 64 bits.
Tolerances: tree_plain.norm_bound; copied values and untouched memory bit for bit."""
import numpy as np
import pytest

import aqueduct as aq
import paged_plain as P
import tree_plain as T

pytestmark = pytest.mark.gpu
THETA, EPS = 1e7, 1e-6
PAIRS = [("f32", "f32"), ("f32", "f16"), ("f32", "bf16"), ("f16", "f16"), ("bf16", "bf16")]


@pytest.fixture(scope="module")
def ctx():
    return aq.Context(0)


class Weight:
    """hd f32 norm weights on the device, `skip` values into their buffer."""

    def __init__(self, ctx, rng, hd, skip=0):
        self.w = (1.0 + 0.3 * rng.standard_normal(hd)).astype(np.float32)
        self.dev = P.Dev(ctx, np.concatenate([np.zeros(skip, np.float32), self.w]))
        self.at = self.dev.buf.p.value + 4 * skip


def want_of(x, w, pos, dim, layout, scaling=("none", {})):
    y = T.normed(x, w.astype(np.float64), EPS)
    if not dim:
        return y, 1.0
    freq, gain = P.frequencies(dim, THETA, scaling[0], scaling[1].get("factor", 1.0), scaling[1].get("orig_ctx", 0))
    return P.rotate(y, pos, dim, layout, freq, gain), gain


def near(got, x, w, want, t, dim, gain, more=0.0):
    limit = T.norm_bound(x, w.astype(np.float64), EPS, want, t, dim, gain) + more
    off = np.abs(got - want) - limit
    assert np.all(off <= 0), f"at {np.unravel_index(np.argmax(off), off.shape)}: over by {off.max():.3g}"


@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("rows,heads,kv,hd,dim,pad,skip,wskip", [
    (1, 24, 4, 256, 64, 0, 0, 0), (7, 3, 1, 128, 128, 0, 0, 0), (130, 5, 5, 96, 48, 8, 0, 0), (3, 1, 1, 80, 40, 0, 0, 0),
    (9, 2, 2, 22, 10, 1, 3, 0), (33, 40, 8, 64, 2, 0, 0, 0), (5, 3, 2, 256, 256, 0, 1, 1), (4, 2, 1, 2, 2, 0, 0, 0),
    (1400, 32, 8, 128, 128, 0, 0, 0), (1100, 24, 4, 256, 64, 0, 0, 0), (40, 3, 2, 8, 4, 0, 0, 1),
    (900, 300, 9, 16, 16, 0, 0, 0)])
def test_norm_rope(ctx, t, layout, rows, heads, kv, hd, dim, pad, skip, wskip):
    print(f"norm {t} {layout} {rows} x {heads}/{kv} x {hd} of {dim} pad {pad} skip {skip} {wskip}", flush=True)
    rng = np.random.default_rng(rows + hd)
    scaling = ("yarn", {"factor": 8.0, "orig_ctx": 4096}) if rows == 33 else ("none", {})
    rope = aq.Rope(ctx, dim, THETA, layout=layout, scaling=scaling[0], **scaling[1])
    q = P.Rows(ctx, rng.standard_normal((rows, heads, hd)) * 2.5, t, pad, skip)
    k = P.Rows(ctx, rng.standard_normal((rows, kv, hd)) * np.exp(rng.uniform(-8, 8, (rows, kv, 1))), t, pad, skip)
    qw, kw = Weight(ctx, rng, hd, wskip), Weight(ctx, rng, hd, wskip)
    pos = rng.integers(-5, 2 ** 31 - 1 if rows == 7 else 200000, rows).astype(np.int32)
    dpos = P.Dev(ctx, pos)
    qo, ko = (P.Rows(ctx, np.full(x.values().shape, 9.0), t, pad, skip) for x in (q, k))
    aq.qk_norm_rope(ctx, q.heads_struct(), qo.heads_struct(), heads, k.heads_struct(), ko.heads_struct(), kv, hd, rows,
                    qw.at, kw.at, EPS, rope, dpos.buf)
    ctx.sync()
    for x, y, w in ((q, qo, qw), (k, ko, kw)):
        want, gain = want_of(x.values(), w.w, pos, dim, layout, scaling)
        # at positions of 2^31 the angle in 64 bits, on both sides, is right to 2^31 * 2^-52 radians of values below 2^5
        near(y.get(), x.values(), w.w, want, t, dim, gain, 2.0 ** -15 * (rows == 7))
    got = [qo.get(), ko.get()]
    for x, w, h, g in ((q, qw, heads, got[0]), (k, kw, kv, got[1])):  # alone and in place: the same bits
        again = P.Rows(ctx, x.values(), t, pad, skip)
        if x is q:
            aq.qk_norm_rope(ctx, again.heads_struct(), again.heads_struct(), h, None, None, 0, hd, rows, w.at, None, EPS,
                            rope, dpos.buf)
        else:
            aq.qk_norm_rope(ctx, None, None, 0, again.heads_struct(), again.heads_struct(), h, hd, rows, None, w.at, EPS,
                            rope, dpos.buf)
        ctx.sync()
        assert np.array_equal(again.get(), g)


@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows,heads,hd", [(1, 1, 1), (3, 5, 7), (2, 4, 255), (60, 8, 256), (2000, 40, 128)])
def test_norm_alone(ctx, t, rows, heads, hd):
    """Without a rope; rows of zeros stay zeros, and rows of the type's largest values that 32-bit squares hold are normed."""
    print(f"norm alone {t} {rows} x {heads} x {hd}", flush=True)
    rng = np.random.default_rng(hd)
    x = rng.standard_normal((rows, heads, hd))
    x[0, 0] = 0.0
    x[-1, -1] *= {"f32": 1e15, "f16": 1e4, "bf16": 1e15}[t]
    q, w = P.Rows(ctx, x, t), Weight(ctx, rng, hd)
    out = P.Rows(ctx, np.full(x.shape, 9.0), t)
    aq.qk_norm_rope(ctx, q.heads_struct(), out.heads_struct(), heads, None, None, 0, hd, rows, w.at, None, EPS)
    ctx.sync()
    got = out.get()
    want, _ = want_of(q.values(), w.w, None, 0, "half")
    near(got, q.values(), w.w, want, t, 0, 1.0)
    assert np.all(got[0, 0] == 0.0)


@pytest.mark.parametrize("row_t,cache_t", PAIRS)
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("heads,kv,hd,dim,page,pad", [(24, 4, 256, 64, 16, 0), (8, 2, 128, 128, 7, 0), (5, 5, 80, 40, 24, 8),
                                                      (3, 1, 8, 8, 1, 1), (28, 4, 96, 0, 64, 0)])
@pytest.mark.parametrize("far", [False, True])
def test_append(ctx, row_t, cache_t, layout, heads, kv, hd, dim, page, pad, far):
    """Into pages; `far`: rotated by positions that are not the rows' places. A prompt, a token, an empty sequence, one that
    is cut by its table, and rows that belong to none."""
    print(f"append {row_t}/{cache_t} {layout} {heads}/{kv} x {hd} of {dim} page {page} pad {pad} far {far}", flush=True)
    rng = np.random.default_rng(hd + page)
    new, lens = [33, 1, 0, 5], [40, 77, 9, 60]
    pg = P.Paged(ctx, rng, new, lens, kv, hd, page, cache_t, cols=-(-77 // page) if page < 64 else 2, n_rows=sum(new) + 3,
                 layout="heads" if page == 7 else "slots")
    pg.table[3, 58 // page:] = 10 ** 6  # the last sequence's end has no page
    pg.upload()
    rope = aq.Rope(ctx, dim, THETA, layout=layout) if dim else None
    q, k, v = (P.Rows(ctx, rng.standard_normal((pg.rows, h, hd)) * 3, row_t, pad) for h in (heads, kv, kv))
    qo = P.Rows(ctx, np.full((pg.rows, heads, hd), 9.0), row_t, pad)
    qw, kw = Weight(ctx, rng, hd), Weight(ctx, rng, hd)
    cache, batch = pg.structs()
    far = far and rope is not None
    pos = np.zeros(pg.rows, np.int64)
    for s in range(4):
        pos[pg.starts[s]: pg.starts[s + 1]] = lens[s] - new[s] + np.arange(new[s])
    turn = rng.integers(-9, 100000, pg.rows).astype(np.int32) if far else pos
    dturn = P.Dev(ctx, turn.astype(np.int32))
    aq.paged_append_norm(ctx, cache, batch, k.heads_struct(), v.heads_struct(), q.heads_struct(), qo.heads_struct(), heads,
                         qw.at, kw.at, EPS, rope, dturn.buf if far else None)
    ctx.sync()
    n = sum(new)
    want, gain = want_of(q.values()[:n], qw.w, turn[:n], dim, layout)
    got = qo.get()
    near(got[:n], q.values()[:n], qw.w, want, row_t, dim, gain)
    assert np.all(got[n:] == 9.0), "rows behind the last sequence"
    wk, _ = want_of(k.values()[:n], kw.w, turn[:n], dim, layout)
    limit = T.norm_bound(k.values()[:n], kw.w.astype(np.float64), EPS, wk, cache_t, dim)
    keys, vals = pg.pools()
    rest_k, rest_v = pg.k.copy(), pg.v.copy()
    for s in range(4):
        for i in range(new[s]):
            r = int(pg.starts[s]) + i
            at = pg.row_of(s, int(pos[r]))
            if at is None:
                continue
            assert np.all(np.abs(keys[at] - wk[r]) <= limit[r]), (s, i)
            assert np.array_equal(vals[at], P.values(P.store(v.values()[r], cache_t), cache_t)), (s, i)
            rest_k[at], rest_v[at] = keys[at], vals[at]
    assert np.array_equal(rest_k, keys, equal_nan=True) and np.array_equal(rest_v, vals, equal_nan=True)
    # without the queries, and with the queries in place: the same
    aq.paged_append_norm(ctx, cache, batch, k.heads_struct(), v.heads_struct(), None, None, 0, None, kw.at, EPS, rope,
                         dturn.buf if far else None)
    again = P.Rows(ctx, q.values(), row_t, pad)
    aq.paged_append_norm(ctx, cache, batch, k.heads_struct(), v.heads_struct(), again.heads_struct(), again.heads_struct(),
                         heads, qw.at, kw.at, EPS, rope, dturn.buf if far else None)
    ctx.sync()
    k2, v2 = pg.pools()
    assert np.array_equal(k2, keys, equal_nan=True) and np.array_equal(v2, vals, equal_nan=True)
    assert np.array_equal(again.get()[:n], got[:n]) and np.array_equal(again.get()[n:], q.values()[n:])


@pytest.mark.parametrize("row_t,cache_t", PAIRS)
def test_append_of_rows_outside(ctx, row_t, cache_t):
    """Rows before the first sequence's start and past the tensors are left alone; a sequence that begins before position 0
    stores what has a place; many rows take the other launch and give the same."""
    print(f"append outside {row_t}/{cache_t}", flush=True)
    rng = np.random.default_rng(8)
    kv, hd, heads = 2, 64, 4
    new, lens = [20, 900], [15, 1300]
    pg = P.Paged(ctx, rng, new, lens, kv, hd, 16, cache_t)
    pg.starts += 6  # rows 0 .. 5: no sequence's
    pg.rows = 6 + 20 + 890  # the last ten are past the tensors
    pg.upload()
    q, k, v = (P.Rows(ctx, rng.standard_normal((pg.rows, h, hd)), row_t) for h in (heads, kv, kv))
    qo = P.Rows(ctx, np.full((pg.rows, heads, hd), 9.0), row_t)
    w = Weight(ctx, rng, hd)
    rope = aq.Rope(ctx, hd, THETA)
    cache, batch = pg.structs()
    aq.paged_append_norm(ctx, cache, batch, k.heads_struct(), v.heads_struct(), q.heads_struct(), qo.heads_struct(), heads,
                         w.at, w.at, EPS, rope)
    ctx.sync()
    pos = np.concatenate([np.arange(20) - 5, 400 + np.arange(890)])
    want, _ = want_of(q.values()[6:], w.w, pos, hd, "half")
    got = qo.get()
    assert np.all(got[:6] == 9.0)
    near(got[6:], q.values()[6:], w.w, want, row_t, hd, 1.0)
    keys, vals = pg.pools()
    at = [(0, int(p), r) if r < 20 else (1, int(p), r) for r, p in enumerate(pos)]
    wk, _ = want_of(k.values()[6:], w.w, pos, hd, "half")
    limit = T.norm_bound(k.values()[6:], w.w.astype(np.float64), EPS, wk, cache_t, hd)
    for s, p, r in at:
        place = pg.row_of(s, p)
        if place is None:
            continue
        assert np.all(np.abs(keys[place] - wk[r]) <= limit[r])
        pg.k[place], pg.v[place] = keys[place], vals[place]
    assert np.array_equal(pg.k, keys, equal_nan=True) and np.array_equal(pg.v, vals, equal_nan=True)


def test_no_rows(ctx):
    w = Weight(ctx, np.random.default_rng(1), 64)
    x = aq.heads(w.at, aq.F32, 64, 64)
    aq.qk_norm_rope(ctx, x, x, 1, None, None, 0, 64, 0, w.at, None, EPS)
    ctx.sync()
    assert np.array_equal(w.dev.get(), w.w)
