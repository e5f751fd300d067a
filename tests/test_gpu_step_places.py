"""Speculative steps at the ends of what they reach: pools and rows 2^32 bytes and more apart, and page tables in place over
many work-groups as a captured graph, whose lengths and counts each replay takes on from the one before."""
import ctypes as C

import numpy as np
import pytest

import aqueduct as aq
import paged_plain as P
import tree_plain as T
from test_gpu_paged_run import Stream, hip

pytestmark = pytest.mark.gpu
THETA, EPS = 1e6, 1e-6


@pytest.fixture(scope="module")
def ctx():
    return aq.Context(0)


@pytest.mark.parametrize("row_t,cache_t", [("f32", "f16"), ("bf16", "bf16"), ("f32", "f32")])
@pytest.mark.parametrize("new", [[2, 1], [70, 5]])
@pytest.mark.parametrize("far", ["page", "head", "slot"])
def test_offsets_past_32_bits(ctx, row_t, cache_t, new, far):
    """Appended with the norms, attended as trees, the paths kept: the bits of the same batch close together."""
    print(f"far {far} {row_t}/{cache_t} {new}", flush=True)
    rng = np.random.default_rng(14)
    kv, hd, heads, slots = 2, 64, 4, 2 if far == "slot" else 16
    lens = ([30, 3] if far == "slot" else [60, 5]) if new[0] == 2 else [74, 6]
    pages = 60 if far == "slot" else 6
    e, es = P.SIZE[cache_t], P.SIZE[row_t]
    wide = 2 ** 32 // e // 4 * 5
    dense = dict(page_stride=slots * kv * hd, slot_stride=kv * hd, head_stride=hd)
    strides = {"page": dict(page_stride=wide, slot_stride=kv * hd, head_stride=hd),
               "head": dict(page_stride=slots * hd, slot_stride=hd, head_stride=wide),
               "slot": dict(page_stride=kv * hd, slot_stride=wide, head_stride=hd)}[far]
    rows, order = sum(new), rng.permutation(pages).astype(np.int32)
    need = [-(-n // slots) for n in lens]
    most = (5 << 20) // (rows * heads) + 1 if rows > 8 else max(lens)  # bounds with which 16-bit chunks take their own kernel
    table = np.full((2, -(-most // slots)), -1, np.int32)
    table[0, : need[0]], table[1, : need[1]] = order[: need[0]], order[need[0]: sum(need)]
    dev = lambda a: P.Dev(ctx, a)  # noqa: E731
    dlens, dtable = dev(np.array(lens, np.int32)), dev(table)
    starts = dev(np.array([0, new[0], rows], np.int32))
    batch = aq.paged_batch(2, starts.buf, dlens.buf, dtable.buf, table.shape[1], rows, max(new), most)
    first = [n - m for n, m in zip(lens, new)]  # what stands before the trees
    dfirst, all_rows = dev(np.array(first, np.int32)), dev(np.array([0, first[0], sum(first)], np.int32))
    fill = aq.paged_batch(2, all_rows.buf, dfirst.buf, dtable.buf, table.shape[1], sum(first), max(first), max(lens))
    words = -(-max(new) // 32)
    mask = dev(T.pack(T.random_trees(rng, new), words))
    path = np.full((2, 8), -1, np.int32)
    keep = [max(1, min(n - 1, 5)) for n in new]
    for s in range(2):
        path[s, : keep[s]] = np.sort(rng.choice(np.arange(1, new[s]) if new[s] > keep[s] else new[s], keep[s], replace=False))
    dpath, dkeep = dev(path), dev(np.array(keep, np.int32))
    depth = dev(rng.integers(0, 99, rows).astype(np.int32))
    qw, kw = (dev((1 + 0.2 * rng.standard_normal(hd)).astype(np.float32)) for _ in range(2))
    x = {n: rng.standard_normal((c, h, hd)) for n, c, h in (("k0", sum(first), kv), ("v0", sum(first), kv), ("k", rows, kv),
                                                            ("v", rows, kv), ("q", rows, heads))}
    rope = aq.Rope(ctx, hd, THETA)
    got = []
    for st in (dense, strides):
        top = (pages - 1) * st["page_stride"] + (slots - 1) * st["slot_stride"] + (kv - 1) * st["head_stride"] + hd
        k, v = aq.DeviceBuffer(ctx, top * e), aq.DeviceBuffer(ctx, top * e)
        cache = aq.paged_kv(k, v, P.TYPES[cache_t], pages, slots, kv, hd, **st)
        # the rows' stride: past 2^32 bytes for a few rows
        stride = heads * hd if st is dense or rows > 8 else 2 ** 32 // es + 4 * 16
        buf = {n: aq.DeviceBuffer(ctx, ((rows - 1) * stride + heads * hd) * es) for n in ("q", "out")}
        h = {n: aq.heads(b, P.TYPES[row_t], stride, hd) for n, b in buf.items()}
        q = P.store(x["q"], row_t)
        for r in range(rows):
            aq.check(aq.lib().aq_memcpy_htod(ctx.h, C.c_void_p(buf["q"].p.value + r * stride * es), q[r].ctypes.data,
                                             q[r].nbytes))
        r = {n: P.Rows(ctx, x[n], row_t) for n in ("k0", "v0", "k", "v")}
        aq.paged_append_norm(ctx, cache, fill, r["k0"].heads_struct(), r["v0"].heads_struct(), None, None, 0, None, kw.buf, EPS,
                             rope)
        aq.paged_append_norm(ctx, cache, batch, r["k"].heads_struct(), r["v"].heads_struct(), h["q"], h["q"], heads, qw.buf,
                             kw.buf, EPS, rope, depth.buf)
        ws = aq.DeviceBuffer(ctx, aq.paged_attention_workspace(ctx, cache, batch, heads))
        aq.paged_tree_attention(ctx, cache, batch, mask.buf, words, heads, h["q"], h["out"], 0.125, 0, None, ws)
        left = dev(np.zeros(2, np.int32))
        aq.paged_tree_commit(ctx, aq.paged_kv_array([cache]), batch, dpath.buf, dkeep.buf, 8, left.buf)
        ctx.sync()
        out = np.zeros_like(q)
        for i in range(rows):
            aq.check(aq.lib().aq_memcpy_dtoh(ctx.h, out[i].ctypes.data, C.c_void_p(buf["out"].p.value + i * stride * es),
                                             out[i].nbytes))
        pool = np.zeros((2, sum(lens), kv, hd), q.dtype if row_t == cache_t else P.store(np.zeros(1), cache_t).dtype)
        i = 0
        for s in range(2):
            for p in range(lens[s]):
                for head in range(kv):
                    at = (int(table[s, p // slots]) * st["page_stride"] + p % slots * st["slot_stride"] +
                          head * st["head_stride"]) * e
                    for b, y in ((k, pool[0, i, head]), (v, pool[1, i, head])):
                        aq.check(aq.lib().aq_memcpy_dtoh(ctx.h, y.ctypes.data, C.c_void_p(b.p.value + at), y.nbytes))
                i += 1
        got.append((P.values(out, row_t), P.values(pool, cache_t), left.get()))
        for b in (k, v, *buf.values(), ws):
            b.free()
    assert np.all(np.isfinite(got[0][0])) and np.abs(got[0][0]).max() > 0.1 and np.all(np.isfinite(got[0][1]))
    assert got[0][2].tolist() == [f + n for f, n in zip(first, keep)]
    for a, b in zip(*got):
        assert np.array_equal(a, b)
    # the paths' rows stand where they belong
    at = 0
    for s in range(2):
        v0 = P.values(P.store(x["v"], cache_t), cache_t)[sum(new[:s]):]
        for i in range(keep[s]):
            assert np.array_equal(got[0][1][1, at + first[s] + i], v0[path[s, i]])
        at += lens[s]


@pytest.mark.parametrize("n_seq,most", [(40, 900), (700, 60), (2500, 9)])
def test_captured_tables_in_place(ctx, n_seq, most):
    """Lengths, counts and the ring's state written over by the last of many work-groups: replays and eager calls in turn,
    each from what the one before left."""
    print(f"captured tables {n_seq} x {most}", flush=True)
    rng = np.random.default_rng(n_seq)
    page, pool, cols, n_rows = 16, n_seq * (most // 16 + 2), 8 * (most // 16 + 1), n_seq * most
    w = T.Tables(n_seq, cols, pool, page)
    w.ring = rng.permutation(pool).astype(np.int32)
    dev = lambda a: P.Dev(ctx, a)  # noqa: E731
    pages, held, ring, state = dev(w.pages), dev(w.held), dev(w.ring), dev(np.array([0, pool, 0, 0], np.int32))
    lens, new, missing, start = (dev(np.zeros(n, np.int32)) for n in (n_seq, n_seq, n_seq, n_seq + 1))
    pos, slots = dev(np.zeros(n_rows, np.int32)), dev(np.zeros(n_rows, np.int64))
    t = aq.page_tables(n_seq, cols, pool, page, pages.buf, held.buf, ring.buf, state.buf)

    def call(stream=None):
        aq.paged_tables(ctx, t, lens.buf, new.buf, n_rows, start.buf, lens.buf, missing.buf, pos.buf, slots.buf, stream=stream)

    st = Stream()
    graph = st.capture(call)
    at = np.zeros(n_seq, np.int64)
    for step in range(8):
        n = rng.integers(0, most + 1, n_seq)
        n[rng.random(n_seq) < 0.4] = -1
        new.buf.upload(n.astype(np.int32))
        ctx.sync()
        if step % 3 == 2:
            call()
            ctx.sync()
        else:
            st.launch(graph)
            st.sync()
        want = w.step(at, n, n_rows)
        for x, d in zip(want, (start, lens, missing, pos, slots)):
            assert np.array_equal(d.get(), x), step
        assert np.array_equal(held.get(), w.held) and state.get().tolist() == [w.first, w.count, 0, 0]
        assert np.array_equal(pages.get(), w.pages) and np.array_equal(ring.get(), w.ring)
        at = np.asarray(want[1], np.int64)
    hip("hipGraphExecDestroy", graph)
    st.close()
