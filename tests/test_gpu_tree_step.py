"""Speculative steps of a batch as a serving loop runs them: page tables from the lengths, norms and rotation into the pages
at the drafts' depths, attention of the trees, the accepted paths kept, and on from the new lengths; eagerly, as a captured
graph replayed while everything changes, and several at once. Tolerances: tree_plain.norm_bound and paged_plain.bound."""
import numpy as np
import pytest

import aqueduct as aq
import paged_plain as P
import tree_plain as T
from test_gpu_paged_run import Stream, hip

pytestmark = pytest.mark.gpu
PAIRS = [("f32", "f32"), ("f32", "f16"), ("f32", "bf16"), ("f16", "f16"), ("bf16", "bf16")]
THETA, EPS = 1e6, 1e-6


@pytest.fixture(scope="module")
def ctx():
    return aq.Context(0)


class Step:
    """n_seq requests over one pool for each of `layers`; each step has at most `most` rows a request."""

    def __init__(self, ctx, seed, row_t, cache_t, n_seq, most, max_len, layers=2, heads=8, kv=2, hd=128, page=16, window=0):
        self.ctx, self.rng = ctx, np.random.default_rng(seed)
        self.row_t, self.cache_t, self.layers, self.heads, self.kv, self.hd = row_t, cache_t, layers, heads, kv, hd
        self.n_seq, self.most, self.page, self.max_len, self.window = n_seq, most, page, max_len, window
        rng, dev = self.rng, lambda a: P.Dev(ctx, a)
        self.cols = -(-max_len // page)
        self.pages = n_seq * self.cols // 2 + 4
        self.words = -(-most // 32)
        self.rows = n_seq * most
        self.want = T.Tables(n_seq, self.cols, self.pages, page)
        self.want.ring = rng.permutation(self.pages).astype(np.int32)
        w = self.want
        self.d = {"pages": dev(w.pages), "held": dev(w.held), "ring": dev(w.ring), "state": dev(np.array([0, w.count, 0, 0], np.int32)),
                  "before": dev(np.zeros(n_seq, np.int32)), "new": dev(np.zeros(n_seq, np.int32)),
                  "start": dev(np.zeros(n_seq + 1, np.int32)), "len": dev(np.zeros(n_seq, np.int32)),
                  "missing": dev(np.zeros(n_seq, np.int32)), "pos": dev(np.zeros(self.rows, np.int32)),
                  "slots": dev(np.zeros(self.rows, np.int64)), "depth": dev(np.zeros(self.rows, np.int32)),
                  "mask": dev(np.zeros((self.rows, self.words), np.uint32)),
                  "path": dev(np.full((n_seq, most), -1, np.int32)), "m": dev(np.zeros(n_seq, np.int32))}
        nan = P.store(np.full((self.pages, page, kv, hd), np.nan), cache_t)
        self.k, self.v = ([dev(nan) for _ in range(layers)] for _ in range(2))
        self.caches = [aq.paged_kv(k.buf, v.buf, P.TYPES[cache_t], self.pages, page, kv, hd) for k, v in zip(self.k, self.v)]
        self.all = aq.paged_kv_array(self.caches)
        self.tables = aq.page_tables(n_seq, self.cols, self.pages, page, *(self.d[n].buf for n in ("pages", "held", "ring", "state")))
        self.batch = aq.paged_batch(n_seq, self.d["start"].buf, self.d["len"].buf, self.d["pages"].buf, self.cols, self.rows, most,
                                    max_len)
        self.ws = aq.DeviceBuffer(ctx, aq.paged_attention_workspace(ctx, self.caches[0], self.batch, heads))
        self.rope = aq.Rope(ctx, hd, THETA)
        self.freq, _ = P.frequencies(hd, THETA)
        self.w = [(1 + 0.2 * rng.standard_normal(hd)).astype(np.float32) for _ in range(2)]
        self.dw = [dev(x) for x in self.w]
        zeros = lambda h: P.Rows(ctx, np.zeros((self.rows, h, hd)), row_t)  # noqa: E731
        self.x = [{n: zeros(h) for n, h in (("q", heads), ("k", kv), ("v", kv))} for _ in range(layers)]
        self.out = [P.Rows(ctx, np.full((self.rows, heads, hd), 9.0), row_t) for _ in range(layers)]
        self.turned = [zeros(heads) for _ in range(layers)]
        self.scale = float(np.float32(hd ** -0.5))
        self.lens = np.zeros(n_seq, np.int64)
        self.kept = {}  # (layer, sequence, position) -> key, its bound, value

    def prepare(self, new):
        """This step's requests, trees, accepted paths and rows, uploaded."""
        rng, up = self.rng, lambda n, a: self.d[n].buf.upload(np.ascontiguousarray(a))
        self.new = np.array(new)
        n = np.maximum(self.new, 0)
        self.used = int(n.sum())
        self.masks = T.random_trees(rng, n, near=2.0)
        depth = np.zeros(self.rows, np.int32)
        depth[: self.used] = [int(m.sum()) - 1 for m in self.masks]
        self.depth = depth
        starts = np.concatenate([[0], np.cumsum(n)])
        path, m = np.full((self.n_seq, self.most), -1, np.int32), np.zeros(self.n_seq, np.int32)
        for s in range(self.n_seq):
            if n[s]:  # the ancestors of some row
                at = np.nonzero(self.masks[int(starts[s]) + int(rng.integers(0, n[s]))])[0]
                path[s, : len(at)], m[s] = at, len(at)
        self.path, self.m = path, m
        for name, a in (("new", self.new.astype(np.int32)), ("depth", depth), ("path", path), ("m", m),
                        ("mask", T.pack(self.masks + [np.zeros(1, bool)] * (self.rows - self.used), self.words))):
            up(name, a)
        for x, out, turned in zip(self.x, self.out, self.turned):
            for r in x.values():
                whole = np.full(r.whole.shape, 7.0).reshape(self.rows, r.heads, self.hd)
                whole[: self.used] = rng.standard_normal((self.used, r.heads, self.hd)) * 2
                r.whole = P.store(whole.reshape(-1), self.row_t)
                r.dev.buf.upload(r.whole)
            out.dev.buf.upload(out.whole)
            turned.dev.buf.upload(turned.whole)

    def call(self, stream=None, ws=None):
        ctx, d = self.ctx, self.d
        aq.paged_tables(ctx, self.tables, d["before"].buf, d["new"].buf, self.rows, d["start"].buf, d["len"].buf, d["missing"].buf,
                        d["pos"].buf, d["slots"].buf, d["depth"].buf, stream=stream)
        for cache, x, out, turned in zip(self.caches, self.x, self.out, self.turned):
            h = {n: r.heads_struct() for n, r in x.items()}
            aq.paged_append_norm(ctx, cache, self.batch, h["k"], h["v"], h["q"], turned.heads_struct(), self.heads, self.dw[0].buf,
                                 self.dw[1].buf, EPS, self.rope, d["pos"].buf, stream=stream)
            aq.paged_tree_attention(ctx, cache, self.batch, d["mask"].buf, self.words, self.heads, turned.heads_struct(),
                                    out.heads_struct(), self.scale, self.window, None, ws or self.ws, stream=stream)
        aq.paged_tree_commit(ctx, self.all, self.batch, d["path"].buf, d["m"].buf, self.most, d["before"].buf, stream=stream)

    def bits(self):
        return [x.dev.get().view(np.uint8) for x in self.out] + [x.get().view(np.uint8) for x in self.k + self.v] + \
               [self.d[n].get() for n in ("pages", "held", "ring", "state", "before", "start", "len", "missing", "pos", "slots")]

    def check(self):
        n = np.maximum(self.new, 0)
        start, length, missing, pos, slots = self.want.step(self.lens, self.new, self.rows, self.depth)
        for name, x in (("start", start), ("len", length), ("missing", missing), ("pos", pos), ("slots", slots),
                        ("pages", self.want.pages), ("held", self.want.held), ("ring", self.want.ring)):
            assert np.array_equal(self.d[name].get(), x), name
        assert np.all(missing == 0), "the test's own pool is too small"
        u = self.used
        base = length - n
        for s in range(self.n_seq):
            if self.new[s] < 0:
                self.kept = {at: x for at, x in self.kept.items() if at[1] != s}
        for layer in range(self.layers):
            x = self.x[layer]
            y = {name: P.rotate(T.normed(x[name].values()[:u], w.astype(np.float64), EPS), pos[:u], self.hd, "half", self.freq)
                 for name, w in (("q", self.w[0]), ("k", self.w[1]))}
            got_q = self.turned[layer].get()
            assert np.all(np.abs(got_q[:u] - y["q"]) <= T.norm_bound(x["q"].values()[:u], self.w[0].astype(np.float64), EPS, y["q"],
                                                                     self.row_t, self.hd))
            limit = T.norm_bound(x["k"].values()[:u], self.w[1].astype(np.float64), EPS, y["k"], self.cache_t, self.hd)
            vals = P.values(P.store(x["v"].values()[:u], self.cache_t), self.cache_t)
            # the pages as the attention saw them: every kept row where it belongs, and this step's rows
            pg = P.Paged.__new__(P.Paged)
            shape = (self.pages, self.page, self.kv, self.hd)
            now_k, now_v = (P.values(d[layer].get().reshape(shape), self.cache_t) for d in (self.k, self.v))
            pg.__dict__.update(kv=self.kv, new=[int(i) for i in n], lens=[int(i) for i in length], starts=start, table=self.want.pages,
                               page=self.page, cols=self.cols, max_len=self.max_len, k=np.full(shape, np.nan), v=np.full(shape, np.nan))
            tree = {}
            for (lay, s, p), (key, lim, val) in self.kept.items():
                if lay == layer and p < base[s]:
                    at = pg.row_of(s, p)
                    assert np.all(np.abs(now_k[at] - key) <= lim) and np.array_equal(now_v[at], val), (layer, s, p)
                    pg.k[at], pg.v[at] = now_k[at], now_v[at]
            for s in range(self.n_seq):
                for i in range(int(n[s])):
                    r = int(start[s]) + i
                    at = pg.row_of(s, int(base[s]) + i)
                    tree[s, i] = at
                    pg.k[at], pg.v[at] = y["k"][r], vals[r]
            # the keys that the attention read: a row's own in its place, or where the commit moved it; those of rows that the
            # commit wrote over are known to their bound only
            lost = 0.0
            for s in range(self.n_seq):
                moved = {int(self.path[s, i]): i for i in range(int(self.m[s]))}
                for j, i in moved.items():
                    at = tree[s, i]
                    assert np.all(np.abs(now_k[at] - y["k"][int(start[s]) + j]) <= limit[int(start[s]) + j]), (layer, s, i, j)
                    assert np.array_equal(now_v[at], vals[int(start[s]) + j])
                    pg.k[tree[s, j]] = now_k[at]
                for i in range(int(self.m[s])):
                    if i not in moved:
                        lost = max(lost, float(limit[int(start[s]) + i].max()))
                for i in range(int(self.m[s]), int(n[s])):  # not written over
                    if i not in moved.values():
                        r = int(start[s]) + i
                        assert np.array_equal(now_v[tree[s, i]], vals[r])
                        assert np.all(np.abs(now_k[tree[s, i]] - y["k"][r]) <= limit[r])
                        if i not in moved:
                            pg.k[tree[s, i]] = now_k[tree[s, i]]
            q = got_q[:u]
            want, parts = T.tree_attention(pg, self.masks, q, self.scale, self.window)
            # a key that is off by `lost`: |q| . lost on its score, twice that on the probabilities
            off_key = np.abs(q).sum(-1, keepdims=True) * lost * self.scale
            bound = P.bound(parts, want, self.row_t, self.cache_t, self.hd) + 2.1 * off_key * parts[0].max(-1, keepdims=True)
            got = self.out[layer].get()
            assert np.all(np.abs(got[:u] - want) <= bound)
            assert np.all(got[u:] == 9.0)
            for s in range(self.n_seq):
                for i in range(int(self.m[s])):
                    r = int(start[s]) + int(self.path[s, i])
                    self.kept[layer, s, int(base[s]) + i] = y["k"][r], limit[r], vals[r]
        self.lens = np.where(self.new < 0, 0, base + self.m)
        assert self.d["before"].get().tolist() == self.lens.tolist()


STEPS = [[20, 9, 0], [7, 8, 5], [1, 40, 1], [0, -1, 12], [12, 30, 0], [-1, 1, 3], [2, 2, 2], [40, 40, 40]]


@pytest.mark.parametrize("row_t,cache_t", PAIRS)
@pytest.mark.parametrize("window", [0, 30])
def test_steps(ctx, row_t, cache_t, window):
    """Requests that come, go on with what is accepted, wait, end and come again: without allocations."""
    s = Step(ctx, 3, row_t, cache_t, 3, 40, 200, window=window)
    before = aq.alloc_counts()
    for new in STEPS:
        print(f"step {row_t}/{cache_t} window {window} new {new}", flush=True)
        s.prepare(new)
        s.call()
        ctx.sync()
        s.check()
    assert aq.alloc_counts() == before


@pytest.mark.parametrize("row_t,cache_t", PAIRS)
@pytest.mark.parametrize("most,max_len", [(40, 200), (8, 1500), (40, 6000)])
def test_captured_steps(ctx, row_t, cache_t, most, max_len):
    """One graph of a whole step replayed as the batch changes, the workspace overwritten and eager steps of a twin between:
    the bits of the eager steps, which are right."""
    print(f"graph {row_t}/{cache_t} most {most} max_len {max_len}", flush=True)
    a, b = (Step(ctx, 4, row_t, cache_t, 3, most, max_len, layers=1) for _ in range(2))
    st = Stream()
    graph = st.capture(a.call)
    for new in STEPS:
        new = [min(n, most) for n in new]
        for s in (a, b):
            s.prepare(new)
            s.ws.upload(np.full(s.ws.nbytes, 0xFF, np.uint8))
        ctx.sync()
        st.launch(graph)
        st.sync()
        b.call()
        ctx.sync()
        for x, y in zip(a.bits(), b.bits()):
            assert np.array_equal(x, y)
        a.check()
        b.lens = a.lens
    hip("hipGraphExecDestroy", graph)
    st.close()


@pytest.mark.parametrize("row_t,cache_t", [("f32", "f16"), ("bf16", "bf16")])
def test_steps_at_once(ctx, row_t, cache_t):
    """Four batches on streams of their own, in flight together, some as graphs."""
    print(f"at once {row_t}/{cache_t}", flush=True)
    ss = [Step(ctx, 20 + i, row_t, cache_t, 3, most, 900, hd=hd, layers=2) for i, (most, hd) in
          enumerate([(8, 128), (40, 64), (40, 128), (12, 256)])]
    streams = [Stream() for _ in ss]
    graphs = [st.capture(s.call) if i % 2 else None for i, (s, st) in enumerate(zip(ss, streams))]
    for new in STEPS[:4]:
        for s in ss:
            s.prepare([min(n, s.most) for n in new])
        ctx.sync()
        for s, st, g in zip(ss, streams, graphs):
            if g is None:
                s.call(stream=st.h.value)
            else:
                st.launch(g)
        for s, st in zip(ss, streams):
            st.sync()
            s.check()
    for st, g in zip(streams, graphs):
        if g is not None:
            hip("hipGraphExecDestroy", g)
        st.close()
