"""Rotary positions and the paged append on the device against their formulas in 64 bits. Tolerances:
paged_plain.rotate_bound; copied values and untouched memory bit for bit."""
import numpy as np
import pytest

import aqueduct as aq
import paged_plain as P

pytestmark = pytest.mark.gpu
THETA = 1e7
SCALINGS = {"none": {}, "linear": {"factor": 4.0}, "yarn": {"factor": 8.0, "orig_ctx": 4096}}


@pytest.fixture(scope="module")
def ctx():
    return aq.Context(0)


def freq_of(dim, scaling):
    kw = SCALINGS[scaling]
    return P.frequencies(dim, THETA, scaling, kw.get("factor", 1.0), kw.get("orig_ctx", 0))


@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("scaling", ["none", "linear", "yarn"])
@pytest.mark.parametrize("rows,heads,hd,dim,pad,skip", [(1, 28, 256, 64, 0, 0), (7, 3, 128, 128, 0, 0), (130, 5, 96, 48, 8, 0),
                                                        (3, 1, 80, 80, 0, 0), (9, 2, 22, 10, 1, 3), (33, 40, 64, 2, 0, 0),
                                                        (600, 9, 128, 96, 0, 0)])
def test_rope(ctx, t, layout, scaling, rows, heads, hd, dim, pad, skip):
    rng = np.random.default_rng(rows + hd)
    rope = aq.Rope(ctx, dim, THETA, layout=layout, scaling=scaling, **SCALINGS[scaling])
    x = P.Rows(ctx, rng.standard_normal((rows, heads, hd)), t, pad, skip)
    pos = rng.integers(-5, 2 ** 31 - 1 if rows == 7 else 200000, rows).astype(np.int32)
    pos[0] = 0
    dpos = P.Dev(ctx, pos)
    freq, gain = freq_of(dim, scaling)
    for inverse in (False, True):
        print(f"rope {t} {layout} {scaling} {rows}x{heads}x{hd} of {dim} pad {pad} skip {skip} inverse {inverse}", flush=True)
        y = P.Rows(ctx, np.full((rows, heads, hd), 9.0), t, pad, skip)
        aq.rope_apply(rope, x.heads_struct(), y.heads_struct(), rows, heads, hd, dpos.buf, inverse)
        ctx.sync()
        want = P.rotate(x.values(), pos, dim, layout, freq, gain, inverse)
        got = y.get()
        # at positions of 2^31 the angle itself, in 64 bits on both sides, is right to 2^31 * 2^-52 radians
        assert np.all(np.abs(got - want) <= P.rotate_bound(x.values(), want, t, gain) + 2.0 ** -20 * (rows == 7))
        assert np.array_equal(got[..., dim:], x.values()[..., dim:])
        again = P.Rows(ctx, x.values(), t, pad, skip)  # in place: the same bits
        aq.rope_apply(rope, again.heads_struct(), again.heads_struct(), rows, heads, hd, dpos.buf, inverse)
        ctx.sync()
        assert np.array_equal(again.get(), got)


@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("scaling", ["none", "yarn"])
def test_inverse_is_the_gradient(ctx, layout, scaling):
    """The gradient of sum(w * rope(x)) is rope's inverse of w: against differences of the device's own outputs, which
    are linear in x, so that a step of any size is exact but for the outputs' rounding (2 x 20 u of values of 4)."""
    rng = np.random.default_rng(3)
    rope = aq.Rope(ctx, 16, THETA, layout=layout, scaling=scaling, **SCALINGS[scaling])
    x, w = rng.standard_normal((2, 2, 1, 20))
    pos = P.Dev(ctx, np.array([3, 1234567], np.int32))

    def apply(v, inverse=False):
        a = P.Rows(ctx, v, "f32")
        aq.rope_apply(rope, a.heads_struct(), a.heads_struct(), 2, 1, 20, pos.buf, inverse)
        ctx.sync()
        return a.get()

    grad = apply(w, True)
    w = P.values(P.store(w, "f32"), "f32")
    base = apply(x)
    for d in range(20):
        step = x.copy()
        step[:, 0, d] = P.values(P.store(x[:, 0, d], "f32"), "f32") + 1.0
        diff = ((apply(step) - base) * w)[:, 0].sum(-1)
        assert np.all(np.abs(diff - grad[:, 0, d]) <= 2 * 20 * 2.0 ** -24 * 6 * np.abs(w).sum())


PAIRS = [("f32", "f32"), ("f32", "f16"), ("f32", "bf16"), ("f16", "f16"), ("bf16", "bf16")]


@pytest.mark.parametrize("row_t,cache_t", PAIRS)
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("heads,kv,hd,dim,page,pool,pad,skip", [
    (24, 4, 256, 64, 16, "slots", 0, 0), (6, 2, 128, 128, 7, "heads", 0, 0), (3, 3, 80, 40, 1, "slots", 1, 1),
    (0, 2, 64, 32, 16, "slots", 0, 0), (0, 5, 8, 0, 32, "heads", 3, 0), (2, 1, 24, 20, 16, "slots", 0, 0)])
@pytest.mark.parametrize("new,lens", [([1, 1, 1], [1, 17, 300]), ([40, 0, 9, 2], [40, 5, 100, 1]), ([700, 801], [900, 801])])
def test_append(ctx, row_t, cache_t, layout, heads, kv, hd, dim, page, pool, pad, skip, new, lens):
    print(f"append {row_t}/{cache_t} {layout} {heads}/{kv} x {hd} of {dim} page {page} {pool} new {new} lens {lens} pad "
          f"{pad} skip {skip}", flush=True)
    rng = np.random.default_rng(hd + sum(new))
    pg = P.Paged(ctx, rng, new, lens, kv, hd, page, cache_t, layout=pool, n_rows=sum(new) + 2)
    n = pg.rows
    k = P.Rows(ctx, rng.standard_normal((n, kv, hd)), row_t, pad, skip)
    v = P.Rows(ctx, rng.standard_normal((n, kv, hd)), row_t, pad, skip)
    rope = aq.Rope(ctx, dim, THETA, layout=layout) if dim else None
    q = qo = None
    if heads:
        q = P.Rows(ctx, rng.standard_normal((n, heads, hd)), row_t, pad, skip)
        qo = P.Rows(ctx, np.full((n, heads, hd), 9.0), row_t, pad, skip)
    cache, batch = pg.structs()
    aq.paged_append(ctx, cache, batch, k.heads_struct(), v.heads_struct(), rope, q.heads_struct() if q else None,
                    qo.heads_struct() if q else None, heads)
    ctx.sync()
    pos = np.concatenate([np.arange(length - a, length) for a, length in zip(new, lens)] + [[0, 0]])
    freq, _ = P.frequencies(dim, THETA) if dim else (None, 1.0)

    def turned(x):
        return P.rotate(x.values(), pos, dim, layout, freq) if dim else x.values()

    want_k, gk = turned(k), pg.k.copy()
    bound_k = P.rotate_bound(k.values(), want_k, cache_t)
    got_k, got_v = pg.pools()
    want_v = pg.v.copy()
    for s, a in enumerate(new):
        for i in range(a):
            r = int(pg.starts[s]) + i
            at = pg.row_of(s, int(pos[r]))
            if at is None:  # the position is negative
                continue
            assert np.all(np.abs(got_k[at] - want_k[r]) <= bound_k[r]), f"key of row {r}"
            if dim < hd:
                assert np.array_equal(got_k[at][:, dim:], P.values(P.store(k.values()[r], cache_t), cache_t)[:, dim:])
            gk[at] = got_k[at]
            want_v[at] = P.values(P.store(v.values()[r], cache_t), cache_t)
    assert np.array_equal(gk, got_k, equal_nan=True), "slots that are not the rows'"
    assert np.array_equal(want_v, got_v, equal_nan=True)
    if heads:
        used, want = sum(new), turned(q)
        got = qo.get()
        assert np.all(got[used:] == 9.0)
        assert np.all(np.abs(got - want)[:used] <= P.rotate_bound(q.values(), want, row_t)[:used])


def test_append_stores_nothing_without_a_page(ctx):
    """Negative positions, holes, positions past the table: the pool stays as it is, the queries are turned."""
    rng = np.random.default_rng(4)
    pg = P.Paged(ctx, rng, [4, 3, 2], [2, 60, 40], 2, 64, 16, "bf16", cols=4)
    pg.table[1, 3] = pg.k.shape[0] + 5  # positions 48 .. 63
    pg.table[2, 2] = -1                 # positions 32 .. 47
    pg.upload()
    k = P.Rows(ctx, rng.standard_normal((9, 2, 64)), "bf16")
    q = P.Rows(ctx, rng.standard_normal((9, 4, 64)), "bf16")
    rope = aq.Rope(ctx, 64, THETA)
    cache, batch = pg.structs()
    aq.paged_append(ctx, cache, batch, k.heads_struct(), k.heads_struct(), rope, q.heads_struct(), q.heads_struct(), 4)
    ctx.sync()
    got_k, got_v = pg.pools()
    pos = np.array([-2, -1, 0, 1, 57, 58, 59, 38, 39])
    freq, _ = P.frequencies(64, THETA)
    want_v = pg.v.copy()
    for r in (2, 3):
        want_v[pg.row_of(0, int(pos[r]))] = k.values()[r]
    assert np.array_equal(want_v, got_v, equal_nan=True)
    assert np.array_equal(np.isnan(pg.k), np.isnan(got_k))
    want = P.rotate(k.values()[2:4], pos[2:4], 64, "half", freq)
    for i in range(2):
        assert np.all(np.abs(got_k[pg.row_of(0, i)] - want[i]) <= P.rotate_bound(k.values()[2 + i], want[i], "bf16"))
    whole = np.random.default_rng(4)  # the queries' own values again
    assert np.all(np.isfinite(q.get()))
