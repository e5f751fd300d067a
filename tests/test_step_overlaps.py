"""Outputs of the page tables and of accepted paths that lie over another array of the call, in whole or in part, caches given
twice, and arrays off their alignment are refused, with their codes and texts, before anything touches a device (no GPU
needed)."""
import pytest

import aqueduct as aq
from test_paged_refusals import FakeCtx, FakeRope, good_batch, good_kv, refused, rows

N_SEQ, COLS, POOL, ROWS = 5, 8, 64, 20
WORDS = {"pages": N_SEQ * COLS, "held": N_SEQ, "held_out": N_SEQ, "free_pages": POOL, "free_state": 4, "free_state_out": 4,
         "kv_before": N_SEQ, "n_new": N_SEQ, "row_start": N_SEQ + 1, "kv_len": N_SEQ, "missing": N_SEQ, "pos": ROWS,
         "slots": 2 * ROWS, "row_depth": ROWS}
READ = {"held", "free_state", "kv_before", "n_new", "row_depth"}
IN_PLACE = {("held", "held_out"), ("free_state", "free_state_out"), ("kv_before", "kv_len")}
AT = {name: 0x10000 + 0x1000 * i for i, name in enumerate(WORDS)}  # never read: every call here is refused


@pytest.mark.parametrize("a", sorted(WORDS))
def test_tables(a):
    """Array `a` over the first and over the last bytes of each other, and at the same place."""
    for b in sorted(WORDS):
        if a == b or (a in READ and b in READ):
            continue
        step = 8 if "slots" in (a, b) else 4
        for at in (AT[b], AT[b] + 4 * WORDS[b] - step, AT[b] - 4 * WORDS[a] + step):
            if at == AT[b] and ((a, b) in IN_PLACE or (b, a) in IN_PLACE):
                continue
            at -= at % step
            x = dict(AT, **{a: at})
            t = aq.page_tables(N_SEQ, COLS, POOL, 16, *(x[n] for n in ("pages", "held", "free_pages", "free_state", "held_out",
                                                                       "free_state_out")))
            refused(aq.AQ_EINVAL, "lies over", aq.paged_tables, FakeCtx(), t, x["kv_before"], x["n_new"], ROWS,
                    *(x[n] for n in ("row_start", "kv_len", "missing", "pos", "slots", "row_depth")))


def test_commit():
    """The lengths over the first and the last bytes of what the call reads; one cache given twice, also as another's values."""
    n, cols, most = 5, 8, 6
    words = {"row_start": n + 1, "kv_len": n, "pages": n * cols, "path": n * most, "path_len": n}
    at = {name: 0x10000 + 0x1000 * i for i, name in enumerate(words)}
    batch = good_batch(n_seq=n, max_pages=cols, n_rows=20, max_rows=9, **{x: at[x] for x in ("row_start", "kv_len", "pages")})
    pools = [good_kv(k=0x100000 + 0x20000 * i, v=0x110000 + 0x20000 * i) for i in range(3)]

    def go(text, kvs, out):
        refused(aq.AQ_EINVAL, text, aq.paged_tree_commit, FakeCtx(), aq.paged_kv_array(kvs), batch, at["path"], at["path_len"],
                most, out)

    for name, size in words.items():
        for out in (at[name], at[name] + 4 * size - 4, at[name] - 4 * n + 4):
            go("lies over", pools, out)
    same = good_kv(k=pools[0].k, v=0x300000)
    crossed = good_kv(k=0x300000, v=pools[1].k)
    for kvs in ([pools[0], pools[1], pools[0]], [*pools, same], [*pools, crossed], [good_kv(k=0x300000, v=0x300000)]):
        go("same memory", kvs, None)


def test_arrays_off_their_alignment():
    """Positions and the batch's arrays, each 2 bytes off, in every call that takes them."""
    ctx = FakeCtx()
    rope, x, y, at = FakeRope(ctx, 64), rows(heads=4), rows(heads=4, data=0x40000), 0x10000

    def go(call, **kw):
        refused(aq.AQ_EINVAL, "is not aligned to its type", call, ctx, **kw)

    go(aq.qk_norm_rope, q=x, q_out=y, n_head=4, k=None, k_out=None, n_head_kv=0, head_dim=64, n_rows=3, q_weight=at, k_weight=None,
       eps=1e-6, rope=rope, pos=at + 2)
    go(aq.paged_append_norm, kv=good_kv(), batch=good_batch(), k=rows(), v=rows(), q=None, q_out=None, n_head=0, q_weight=None,
       k_weight=at, eps=1e-6, rope=rope, pos=at + 2)
    refused(aq.AQ_EINVAL, "is not aligned to its type", aq.rope_apply, rope, x, y, 3, 4, 64, at + 2)
    for name in ("row_start", "kv_len", "pages"):
        b = good_batch(**{name: at + 2})
        go(aq.paged_append, kv=good_kv(), batch=b, k=rows(), v=rows())
        go(aq.paged_append_norm, kv=good_kv(), batch=b, k=rows(), v=rows(), q=None, q_out=None, n_head=0, q_weight=None,
           k_weight=at, eps=1e-6)
        go(aq.paged_attention, kv=good_kv(), batch=b, n_head=4, q=x, out=y, scale=0.1, workspace=at, workspace_bytes=1 << 30)
        go(aq.paged_tree_attention, kv=good_kv(), batch=b, mask=at, mask_words=1, n_head=4, q=x, out=y, scale=0.1, workspace=at,
           workspace_bytes=1 << 30)
        go(aq.paged_tree_commit, kvs=good_kv(v=0x80000), batch=b, path=at, path_len=at, max_path=4)
