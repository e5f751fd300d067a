"""The calls of a speculative step over pages where their arguments end: heads that leave lanes of a wave without one. Against
the definitions in 64 bits; tolerances: tree_plain.norm_bound and paged_plain.bound, by arithmetic."""
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
