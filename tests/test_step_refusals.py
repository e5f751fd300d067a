"""What the calls of a speculative step over pages refuse, with their codes and texts: the head norms with the rotation, tree
attention, accepted paths, page tables. Every refusal comes before anything touches a device (no GPU needed)."""
import pytest

import aqueduct as aq
from test_paged_refusals import FAKE, FakeCtx, FakeRope, good_batch, good_kv, refused, rows


@pytest.fixture()
def ctx():
    return FakeCtx()


FAR = 2 * FAKE


def test_qk_norm_rope(ctx):
    rope = FakeRope(ctx, 64)

    def go(code, text, **kw):
        a = dict(q=rows(heads=4), q_out=rows(heads=4, data=FAR), n_head=4, k=rows(), k_out=rows(data=FAR), n_head_kv=2, head_dim=64,
                 n_rows=3, q_weight=FAKE, k_weight=FAKE, eps=1e-6, rope=rope, pos=FAKE)
        a.update(kw)
        refused(code, text, aq.qk_norm_rope, ctx, **a)

    go(aq.AQ_EINVAL, "neither", q=None, q_out=None, k=None, k_out=None)
    go(aq.AQ_EINVAL, "go together", q_out=None)
    go(aq.AQ_EINVAL, "go together", k=None)
    go(aq.AQ_EINVAL, "size", n_head=0)
    go(aq.AQ_EINVAL, "size", n_head_kv=70000)
    go(aq.AQ_EINVAL, "size", n_rows=1 << 24)
    go(aq.AQ_EUNSUP, "head_dim", head_dim=257)
    go(aq.AQ_EUNSUP, "head_dim", head_dim=0)
    for eps in (0.0, -1e-6, float("nan"), float("inf")):
        go(aq.AQ_EINVAL, "eps", eps=eps)
    go(aq.AQ_EINVAL, "rotated", head_dim=32)
    go(aq.AQ_EINVAL, "type", q=rows(t=aq.Q4_K, heads=4))
    go(aq.AQ_EINVAL, "different types", q_out=rows(t=aq.BF16, heads=4, data=FAR))
    go(aq.AQ_EINVAL, "different types", k=rows(t=aq.BF16), k_out=rows(t=aq.BF16, data=FAR))
    go(aq.AQ_EINVAL, "null", q=rows(data=None, heads=4))
    go(aq.AQ_EINVAL, "aligned", k=rows(data=FAKE + 1))
    go(aq.AQ_EINVAL, "rows overlap", q=rows(heads=4, row=32))
    go(aq.AQ_EINVAL, "heads overlap", k_out=rows(data=FAR, head=32))
    go(aq.AQ_EINVAL, "in place", q_out=rows(heads=4, row=300))
    go(aq.AQ_EINVAL, "q_weight", q_weight=None)
    go(aq.AQ_EINVAL, "k_weight", k_weight=FAKE + 2)
    go(aq.AQ_EINVAL, "positions go together", pos=None)
    go(aq.AQ_EINVAL, "positions go together", rope=None)
    other = FakeCtx()
    other.mem[0] = 1
    go(aq.AQ_EINVAL, "another device", rope=FakeRope(other, 64))
    odd = dict(heads=1, hd=65)
    go(aq.AQ_EINVAL, "odd", q=rows(**odd), q_out=rows(data=FAR, **odd), n_head=1, k=None, k_out=None, head_dim=65,
       rope=FakeRope(ctx, 64, layout=1))


def test_append_norm(ctx):
    rope = FakeRope(ctx, 64)

    def go(code, text, **kw):
        a = dict(kv=good_kv(), batch=good_batch(), k=rows(), v=rows(), q=rows(heads=4), q_out=rows(heads=4, data=FAR), n_head=4,
                 q_weight=FAKE, k_weight=FAKE, eps=1e-6, rope=rope, pos=FAKE)
        a.update(kw)
        refused(code, text, aq.paged_append_norm, ctx, **a)

    go(aq.AQ_EINVAL, "null", kv=None)
    go(aq.AQ_EINVAL, "null", k=None)
    go(aq.AQ_EINVAL, "eps", eps=0.0)
    go(aq.AQ_EINVAL, "k_weight", k_weight=None)
    go(aq.AQ_EINVAL, "q_weight", q_weight=None)
    go(aq.AQ_EINVAL, "go together", q_out=None)
    go(aq.AQ_EINVAL, "n_head", n_head=0)
    go(aq.AQ_EINVAL, "k and v of different types", v=rows(t=aq.F32))
    go(aq.AQ_EINVAL, "F32 or of the cache's type", k=rows(t=aq.BF16), v=rows(t=aq.BF16))
    go(aq.AQ_EINVAL, "q and k of different types", q=rows(t=aq.F32, heads=4), q_out=rows(t=aq.F32, heads=4, data=FAR))
    go(aq.AQ_EINVAL, "in place", q_out=rows(heads=4, row=300))
    go(aq.AQ_EINVAL, "positions without a rope", rope=None)
    go(aq.AQ_EINVAL, "rotated", rope=FakeRope(ctx, 66))
    go(aq.AQ_EUNSUP, "head_dim", kv=good_kv(head_dim=60))
    go(aq.AQ_EINVAL, "reaches past", batch=good_batch(max_pages=1 << 28))


def test_tree_attention(ctx):
    def go(code, text, **kw):
        a = dict(kv=good_kv(), batch=good_batch(), mask=FAKE, mask_words=1, n_head=4, q=rows(heads=4), out=rows(heads=4, data=FAR),
                 scale=0.125, workspace=FAKE, workspace_bytes=1 << 30)
        a.update(kw)
        refused(code, text, aq.paged_tree_attention, ctx, **a)

    go(aq.AQ_EINVAL, "null", batch=None)
    go(aq.AQ_EINVAL, "null mask", mask=None)
    go(aq.AQ_EINVAL, "mask_dev is not aligned", mask=FAKE + 2)
    go(aq.AQ_EINVAL, "mask of 0 words for 2 rows", mask_words=0)
    go(aq.AQ_EINVAL, "mask of 2 words for 65 rows", mask_words=2, batch=good_batch(n_rows=65, max_rows=65))
    go(aq.AQ_EINVAL, "mask of", mask_words=1 << 20)
    go(aq.AQ_EINVAL, "multiple of n_head_kv", n_head=5)
    go(aq.AQ_EINVAL, "F32 or of the cache's type", q=rows(t=aq.BF16, heads=4))
    go(aq.AQ_EINVAL, "different types", out=rows(t=aq.F32, heads=4, data=FAR))
    go(aq.AQ_EINVAL, "in place", out=rows(heads=4, row=300))
    for scale in (0.0, -1.0, float("nan"), float("inf")):
        go(aq.AQ_EINVAL, "scale", scale=scale)
    go(aq.AQ_EINVAL, "aq_paged_tree_attention: workspace is null", workspace=None)
    go(aq.AQ_EINVAL, "workspace of 16 bytes", workspace_bytes=16)


def test_tree_commit(ctx):
    def go(code, text, **kw):
        a = dict(kvs=aq.paged_kv_array([good_kv(), good_kv(k=FAR, v=FAR)]), batch=good_batch(), path=FAKE, path_len=FAKE, max_path=4,
                 kv_len_out=FAR)
        a.update(kw)
        refused(code, text, aq.paged_tree_commit, ctx, **a)

    go(aq.AQ_EINVAL, "null", kvs=None)
    go(aq.AQ_EINVAL, "null", kvs=aq.paged_kv_array([]))
    go(aq.AQ_EINVAL, "null", batch=None)
    go(aq.AQ_EINVAL, "null path", path=None)
    go(aq.AQ_EINVAL, "null path", path_len=None)
    go(aq.AQ_EINVAL, "null path", max_path=0)
    go(aq.AQ_EINVAL, "max_path", max_path=1 << 24)
    go(aq.AQ_EINVAL, "aligned to its type", path_len=FAKE + 1)
    go(aq.AQ_EINVAL, "lies over", kv_len_out=FAKE)
    go(aq.AQ_EINVAL, "lies over", path=FAR)
    for kw in (dict(type=aq.BF16), dict(n_pages=63), dict(page_size=8), dict(n_head_kv=1, slot_stride=128), dict(slot_stride=256),
               dict(page_stride=1 << 14)):
        go(aq.AQ_EINVAL, "different shapes", kvs=aq.paged_kv_array([good_kv(), good_kv(**kw)]))
    go(aq.AQ_EINVAL, "null k or v", kvs=aq.paged_kv_array([good_kv(), good_kv(v=None)]))


def test_tables(ctx):
    def go(code, text, t=None, **kw):
        a = dict(n_seq=2, max_pages=8, n_pages=64, page_size=16, pages=FAKE, held=FAKE, free_pages=FAKE, free_state=FAKE)
        a.update(t or {})
        b = dict(kv_before=FAKE, n_new=FAR, n_rows=4, row_start=4 * FAKE, kv_len=FAKE + 256, missing=FAR, pos=FAR, slots=FAR)
        b.update(kw)
        refused(code, text, aq.paged_tables, ctx, aq.page_tables(**a), **b)

    go(aq.AQ_EINVAL, "2^24", dict(n_seq=1 << 24))
    go(aq.AQ_EINVAL, "2^24", n_rows=1 << 24)
    for t in (dict(n_pages=0), dict(n_pages=1 << 31), dict(page_size=0)):
        go(aq.AQ_EINVAL, "pages", t)
    go(aq.AQ_EINVAL, "max_pages", dict(max_pages=0))
    go(aq.AQ_EINVAL, "2^31 positions", dict(max_pages=1 << 27))
    go(aq.AQ_EINVAL, "free pages", dict(free_pages=None))
    go(aq.AQ_EINVAL, "free pages", dict(free_state=None))
    go(aq.AQ_EINVAL, "null array", dict(pages=None))
    go(aq.AQ_EINVAL, "null array", dict(held=None))
    for name in ("kv_before", "n_new", "kv_len"):
        go(aq.AQ_EINVAL, "null array", **{name: None})
    go(aq.AQ_EINVAL, "row_start", row_start=None)
    go(aq.AQ_EINVAL, "depths without positions", pos=None, row_depth=FAKE)
    go(aq.AQ_EINVAL, "aligned", slots=FAR + 4)
    go(aq.AQ_EINVAL, "aligned", missing=FAR + 2)
    go(aq.AQ_EINVAL, "lies over", kv_len=FAR)
    go(aq.AQ_EINVAL, "lies over", row_start=FAR)
    go(aq.AQ_EINVAL, "lies over", dict(held_out=FAR))
