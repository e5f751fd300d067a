"""Attention over pages at the ends of the types' ranges: infinite keys at every head size, values near the largest number,
and values that are all the same. Tolerances: paged_plain.bound."""
import numpy as np
import pytest

import aqueduct as aq
import paged_plain as P
from test_gpu_paged_attention import PAIRS, bounds, run

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    return aq.Context(0)


@pytest.mark.parametrize("row_t,cache_t", PAIRS)
@pytest.mark.parametrize("hd", [8, 24, 64, 72, 80, 96, 128, 160, 192, 200, 256])
@pytest.mark.parametrize("new", [1, 40])
@pytest.mark.parametrize("value", [np.inf, -np.inf])
def test_infinite_keys_at_the_end_of_a_head(ctx, row_t, cache_t, hd, new, value):
    """An infinity in a key's last value: a row whose score is plus infinity is NaN, one whose score is minus infinity is as
    if the position were not there, whatever the head's size."""
    print(f"infinite keys {row_t}/{cache_t} head {hd} new {new} {value}", flush=True)
    rng = np.random.default_rng(71)
    pg = P.Paged(ctx, rng, [new], [150], 2, hd, 1, cache_t)
    pg.k[pg.row_of(0, 70)][:, hd - 1] = value
    pg.upload()
    q = P.Rows(ctx, rng.standard_normal((new, 4, hd)), row_t)
    up = q.values()[..., hd - 1] * np.sign(value) > 0
    scale = float(np.float32(hd ** -0.5))
    without = P.Paged.__new__(P.Paged)
    without.__dict__.update(pg.__dict__, table=pg.table.copy())
    without.table[0, 70] = -1  # its page is its own
    want, parts = P.attention(without, q.values(), scale)
    limit = P.bound(parts, want, row_t, cache_t, hd)
    for loose in bounds(pg, q):
        out = P.Rows(ctx, np.full((new, 4, hd), 9.0), row_t)
        run(ctx, pg, q, out, scale, loose=loose)
        got = out.get()
        assert np.array_equal(np.isnan(got).all(-1), up) and np.array_equal(np.isnan(got).any(-1), up)
        assert np.all((np.abs(got - want) <= limit)[~up])


@pytest.mark.parametrize("row_t,cache_t", PAIRS)
@pytest.mark.parametrize("hd", [64, 128, 200, 256])
@pytest.mark.parametrize("new", [1, 40])
def test_values_near_the_largest_number(ctx, row_t, cache_t, hd, new):
    """Scores that rise by e^4 after the first tiles, over values whose sum is still finite: no weight is above 1 on the way.
    At positions from 128 on (22 of them) the value is `big`: their sum, 22 big, is below the type's largest number."""
    print(f"large values {row_t}/{cache_t} head {hd} new {new}", flush=True)
    rng = np.random.default_rng(72)
    pg = P.Paged(ctx, rng, [new], [150], 2, hd, 16, cache_t)
    big = 2000.0 if cache_t == "f16" else 1e37
    for p in range(150):
        at = pg.row_of(0, p)
        pg.k[at] = 4.0 if p >= 128 else 0.0
        if p >= 128:
            pg.v[at] = big * rng.choice([-1.0, 1.0], (2, hd))
    pg.upload()
    q = P.Rows(ctx, np.ones((new, 4, hd)), row_t)
    scale = 1.0 / hd if hd != 200 else float(np.float32(1.0 / hd))
    want, parts = P.attention(pg, q.values(), scale)
    limit = P.bound(parts, want, row_t, cache_t, hd)
    for loose in bounds(pg, q):
        out = P.Rows(ctx, np.full((new, 4, hd), 9.0), row_t)
        run(ctx, pg, q, out, scale, loose=loose)
        got = out.get()
        assert np.all(np.isfinite(got)) and np.all(np.abs(got - want) <= limit)


@pytest.mark.parametrize("row_t,cache_t", PAIRS)
@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("new", [1, 4, 40])
def test_equal_values_come_out_as_they_are(ctx, row_t, cache_t, hd, new):
    """A mean of equal values is that value, however the weights are rounded: what the values are summed with is what they
    are divided by. One position of 16 has weight 1, the others just over half a step of the cache's type above 1/2: their
    roundings all go one way, by 0.87 half steps of the sum, where half a step of a number just below 2 is 0.5 of that.
    f32 rows keep weights to 2^-21 (paged_plain.bound)."""
    print(f"equal values {row_t}/{cache_t} head {hd} new {new}", flush=True)
    rng = np.random.default_rng(73)
    pg = P.Paged(ctx, rng, [new], [150], 2, hd, 16, cache_t)
    step = P.HALF_STEP[cache_t]
    value = 2.0 - 4 * step
    pg.k[:], pg.v[:] = 0.0, value
    for p in range(0, 150, 16):
        pg.k[pg.row_of(0, p)][:, 0] = 1.0
    pg.upload()
    x = np.zeros((new, 4, hd))
    x[..., 0] = 1.0
    q = P.Rows(ctx, x, row_t)
    weight = 0.5 * (1.0 + step * 1.01)  # of two neighbours 0.5 and 0.5 (1 + 2 step), nearer to the second
    scale = float(np.float32(-np.log(weight)))
    want, parts = P.attention(pg, q.values(), scale)
    limit = P.bound(parts, want, row_t, cache_t, hd)
    for loose in bounds(pg, q):
        out = P.Rows(ctx, np.full((new, 4, hd), 9.0), row_t)
        run(ctx, pg, q, out, scale, loose=loose)
        if row_t == "f32":
            assert np.all(np.abs(out.get() - value) <= limit)
        else:
            assert np.all(out.get() == value)


@pytest.mark.parametrize("t,new,length,nats", [("f16", 1, 300000, 20.0), ("f16", 4, 300000, 20.0), ("f16", 40, 20000, 15.0),
                                               ("bf16", 1, 20000, 10.0), ("bf16", 40, 20000, 10.0)])
def test_long_tails_weigh_in_sum_and_values_alike(ctx, t, new, length, nats):
    """One position of weight 1 and a long rest of weights that are subnormal numbers where f16 probabilities are kept (2^14
    times their size, of many rows 2^7 times): the sum takes them as the product does. The rest's share, at least 6e-4, is
    more than half a step of the output."""
    print(f"long tails {t} new {new} length {length}", flush=True)
    pg = P.Paged(ctx, np.random.default_rng(74), [new], [length], 1, 64, 64, t)
    value = 2.0 - 4 * P.HALF_STEP[t]
    pg.k[:], pg.v[:] = 0.0, value
    pg.k[pg.row_of(0, 0)][:, 0] = 1.0
    pg.upload()
    x = np.zeros((new, 1 if new < 40 else 2, 64))
    x[..., 0] = nats
    q = P.Rows(ctx, x, t)
    for loose in bounds(pg, q):
        out = P.Rows(ctx, np.full(x.shape, 9.0), t)
        run(ctx, pg, q, out, 1.0, loose=loose)
        assert np.all(out.get() == value), np.unique(out.get())
