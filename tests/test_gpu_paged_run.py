"""The rotary and paged operators as a serving loop uses them: append and attend over many steps, captured graphs replayed
while lengths, tables and rows change, calls at once on streams of their own, pools and rows past 32-bit offsets, batches
of more row tiles than one work-group divides, and what the library allocates meanwhile (nothing)."""
import ctypes as C

import numpy as np
import pytest

import aqueduct as aq
import paged_plain as P

pytestmark = pytest.mark.gpu
PAIRS = [("f32", "f32"), ("f32", "f16"), ("f32", "bf16"), ("f16", "f16"), ("bf16", "bf16")]
THETA = 1e6


@pytest.fixture(scope="module")
def ctx():
    return aq.Context(0)


def hip(name, *args):
    rc = getattr(aq.lib(), name)(*args)
    assert rc == 0, f"{name}: {rc}"


class Stream:
    def __init__(self):
        self.h = C.c_void_p()
        hip("hipStreamCreateWithFlags", C.byref(self.h), 1)  # does not wait for the null stream

    def sync(self):
        hip("hipStreamSynchronize", self.h)

    def capture(self, calls):
        """A graph of what calls(stream) queues."""
        graph, run = C.c_void_p(), C.c_void_p()
        hip("hipStreamBeginCapture", self.h, 0)
        try:
            calls(self.h.value)
        finally:
            hip("hipStreamEndCapture", self.h, C.byref(graph))
        hip("hipGraphInstantiate", C.byref(run), graph, None, None, C.c_size_t(0))
        hip("hipGraphDestroy", graph)
        return run

    def launch(self, graph):
        hip("hipGraphLaunch", graph, self.h)

    def close(self):
        hip("hipStreamDestroy", self.h)


class Serving:
    """A batch whose rows, lengths and tables change in place between steps, with append and attention over it."""

    def __init__(self, ctx, seed, row_t, cache_t, n_seq, most, max_len, heads=8, kv=2, hd=128, page=16, gated=True, window=0):
        self.ctx, self.rng = ctx, np.random.default_rng(seed)
        self.row_t, self.cache_t, self.heads, self.kv, self.hd, self.page = row_t, cache_t, heads, kv, hd, page
        self.n_seq, self.most, self.max_len, self.window = n_seq, most, max_len, window
        self.cols = -(-max_len // page)
        self.pages = n_seq * self.cols + 3
        self.k, self.v = (P.Dev(ctx, P.store(np.full((self.pages, page, kv, hd), np.nan), cache_t)) for _ in range(2))
        self.rows = n_seq * most
        self.rope = aq.Rope(ctx, hd, THETA)
        self.freq, _ = P.frequencies(hd, THETA)
        self.order = self.rng.permutation(self.pages)
        self.table = np.full((n_seq, self.cols), -1, np.int32)
        self.starts, self.lens = np.zeros(n_seq + 1, np.int32), np.zeros(n_seq, np.int32)
        self.dtable, self.dstarts, self.dlens = (P.Dev(ctx, a) for a in (self.table, self.starts, self.lens))
        self.x = {n: P.Rows(ctx, np.zeros((self.rows, h, hd)), row_t) for n, h in
                  (("q", heads), ("k", kv), ("v", kv), ("gate", heads))}
        self.turned = P.Rows(ctx, np.zeros((self.rows, heads, hd)), row_t)
        self.out = P.Rows(ctx, np.full((self.rows, heads, hd), 9.0), row_t)
        self.gated = gated
        self.cache = aq.paged_kv(self.k.buf, self.v.buf, P.TYPES[cache_t], self.pages, page, kv, hd)
        self.batch = aq.paged_batch(n_seq, self.dstarts.buf, self.dlens.buf, self.dtable.buf, self.cols, self.rows, most,
                                    max_len)
        self.ws = aq.DeviceBuffer(ctx, aq.paged_attention_workspace(ctx, self.cache, self.batch, heads))
        self.scale = float(np.float32(hd ** -0.5))
        self.want = {}  # (sequence, position) -> its rotated key and its value, 64 bits

    def step(self, new):
        """Room, rows and lengths for new[s] more positions of each sequence."""
        self.new = list(new)
        self.starts[1:] = np.cumsum(new)
        self.lens += np.array(new, np.int32)
        for s in range(self.n_seq):
            n = -(-int(self.lens[s]) // self.page)
            self.table[s, :n] = self.order[s * self.cols: s * self.cols + n]
        for name, r in self.x.items():
            whole = np.full(r.whole.shape, 7.0)
            self.used = int(self.starts[-1])
            v = whole.reshape(self.rows, r.heads, self.hd)
            v[: self.used] = self.rng.standard_normal((self.used, r.heads, self.hd))
            r.whole = P.store(whole, self.row_t)
            r.dev.buf.upload(r.whole)
        self.pos = np.concatenate([np.arange(self.lens[s] - n, self.lens[s]) for s, n in enumerate(new)]).astype(np.int64)
        self.seq = np.repeat(np.arange(self.n_seq), new)
        self.out.dev.buf.upload(self.out.whole)
        self.turned.dev.buf.upload(self.turned.whole)
        for d, a in ((self.dtable, self.table), (self.dstarts, self.starts), (self.dlens, self.lens)):
            d.buf.upload(a)
        k, v = self.x["k"].values()[: self.used], self.x["v"].values()[: self.used]
        turned = P.rotate(k, self.pos, self.hd, "half", self.freq)
        limit = P.rotate_bound(k, turned, self.cache_t)
        for r in range(self.used):
            self.want[int(self.seq[r]), int(self.pos[r])] = turned[r], limit[r], P.values(P.store(v[r], self.cache_t),
                                                                                          self.cache_t)

    def call(self, stream=None, ws=None):
        h = {n: r.heads_struct() for n, r in self.x.items()}
        aq.paged_append(self.ctx, self.cache, self.batch, h["k"], h["v"], self.rope, h["q"], self.turned.heads_struct(),
                        self.heads, stream=stream)
        aq.paged_attention(self.ctx, self.cache, self.batch, self.heads, self.turned.heads_struct(),
                           self.out.heads_struct(), self.scale, self.window, h["gate"] if self.gated else None,
                           self.ws if ws is None else ws, stream=stream)

    def bits(self):
        return self.out.dev.get().view(np.uint8)

    def check(self):
        """Every row ever appended is where it belongs; this step's outputs are the attention over them."""
        pg = P.Paged.__new__(P.Paged)
        shape = (self.pages, self.page, self.kv, self.hd)
        pg.k, pg.v = (P.values(d.get().reshape(shape), self.cache_t) for d in (self.k, self.v))
        pg.__dict__.update(kv=self.kv, new=self.new, lens=self.lens, starts=self.starts, table=self.table, page=self.page,
                           cols=self.cols, max_len=self.max_len)
        for (s, p), (k, limit, v) in self.want.items():
            at = pg.row_of(s, p)
            assert np.all(np.abs(pg.k[at] - k) <= limit), (s, p)
            assert np.array_equal(pg.v[at], v), (s, p)
        n = self.used
        x = self.x["q"].values()[:n]
        turned = P.rotate(x, self.pos, self.hd, "half", self.freq)
        q = self.turned.get()
        assert np.all(np.abs(q[:n] - turned) <= P.rotate_bound(x, turned, self.row_t))
        assert np.all(q[n:] == 0.0)
        gate = self.x["gate"].values()[:n] if self.gated else None
        want, parts = P.attention(pg, q[:n], self.scale, self.window, gate)
        got = self.out.get()
        assert np.all(np.abs(got[:n] - want) <= P.bound(parts, want, self.row_t, self.cache_t, self.hd))
        assert np.all(got[n:] == 9.0)


@pytest.mark.parametrize("row_t,cache_t", PAIRS)
@pytest.mark.parametrize("window", [0, 50])
def test_steps_of_a_batch(ctx, row_t, cache_t, window):
    """A prompt, single tokens, drafts to verify, a sequence that waits and one that comes in late: without allocations."""
    s = Serving(ctx, 41, row_t, cache_t, 3, 70, 300, window=window)
    before = aq.alloc_counts()
    for new in ([70, 33, 0], [1, 1, 1], [4, 0, 4], [1, 1, 0], [9, 70, 1], [0, 0, 0], [1, 1, 1]):
        print(f"step {row_t}/{cache_t} window {window} new {new}", flush=True)
        s.step(new)
        s.call()
        ctx.sync()
        s.check()
    assert aq.alloc_counts() == before


@pytest.mark.parametrize("row_t,cache_t", PAIRS)
@pytest.mark.parametrize("most,max_len", [(1, 300), (4, 300), (1, 1500), (4, 1500), (40, 1500), (40, 6000)])
def test_captured_steps(ctx, row_t, cache_t, most, max_len):
    """One graph of append and attention, replayed as the batch changes, with the workspace overwritten and eager calls
    between: each replay gives the bits of the eager call."""
    s, st = Serving(ctx, 42, row_t, cache_t, 3, most, max_len), Stream()
    print(f"graph {row_t}/{cache_t} most {most} max_len {max_len}", flush=True)
    graph = st.capture(s.call)
    other = aq.DeviceBuffer(ctx, s.ws.nbytes)
    junk = np.full(s.ws.nbytes, 0xFF, np.uint8)
    s.lens[:] = [0, min(700, max_len // 2), 20]
    filled = P.store(s.rng.standard_normal((s.pages, s.page, s.kv, s.hd)), cache_t)
    s.k.buf.upload(filled)
    s.v.buf.upload(filled)
    for new in ([1, 1, 1], [most, 0, most], [0, most, 1], [most, most, most], [0, 0, 0]):
        s.step(new)
        s.ws.upload(junk)
        ctx.sync()
        st.launch(graph)
        st.sync()
        got, cache = s.bits(), s.k.get().view(np.uint8)
        s.check()
        s.out.dev.buf.upload(s.out.whole)
        other.upload(junk)
        s.call(ws=other)
        ctx.sync()
        assert np.array_equal(s.bits(), got) and np.array_equal(s.k.get().view(np.uint8), cache)
    hip("hipGraphExecDestroy", graph)
    st.close()


@pytest.mark.parametrize("row_t,cache_t", [("f32", "f32"), ("f32", "f16"), ("bf16", "bf16")])
def test_calls_at_once(ctx, row_t, cache_t):
    """Four batches on streams of their own, eager and as graphs, all in flight together."""
    print(f"at once {row_t}/{cache_t}", flush=True)
    ss = [Serving(ctx, 50 + i, row_t, cache_t, 2, most, 4000, hd=hd) for i, (most, hd) in
          enumerate([(1, 128), (4, 64), (40, 128), (1, 256)])]
    streams = [Stream() for _ in ss]
    graphs = [st.capture(s.call) for s, st in zip(ss, streams)]
    for s in ss:
        x = P.store(s.rng.standard_normal((s.pages, s.page, s.kv, s.hd)), cache_t)
        s.k.buf.upload(x)
        s.v.buf.upload(x)
        s.lens[:] = [3900, 100]
        s.step([s.most, 1])
    ctx.sync()
    for _ in range(5):
        for s, st, g in zip(ss, streams, graphs):
            st.launch(g)
            s.call(stream=st.h.value)
    for st in streams:
        st.sync()
    for s in ss:
        s.check()
    for st, g in zip(streams, graphs):
        hip("hipGraphExecDestroy", g)
        st.close()


@pytest.mark.parametrize("row_t,cache_t", [("f32", "f16"), ("bf16", "bf16"), ("f32", "f32")])
@pytest.mark.parametrize("new", [[2, 1], [70, 5]])
@pytest.mark.parametrize("far", ["page", "head", "slot"])
def test_offsets_past_32_bits(ctx, row_t, cache_t, new, far):
    """A pool whose pages, heads or slots lie 2^32 bytes and more apart, and rows as far: appended, attended, compared with
    the same batch close together, bit for bit."""
    print(f"far {far} {row_t}/{cache_t} {new}", flush=True)
    rng = np.random.default_rng(4)
    kv, hd, heads, slots, pages = 2, 64, 4, {"slot": 2}.get(far, 16), 6
    lens, e = ([60, 5] if new[0] == 2 else [70, 6]), P.SIZE[cache_t]
    if far == "slot":
        lens = [n // 2 if new[0] == 2 else n for n in lens]
        pages = 60
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
    starts, dlens = np.array([0, new[0], rows], np.int32), np.array(lens, np.int32)
    arrays = [P.Dev(ctx, a) for a in (starts, dlens, table)]
    batch = aq.paged_batch(2, *(a.buf for a in arrays), table.shape[1], rows, max(new), most)
    all_rows = P.Dev(ctx, np.array([0, lens[0], sum(lens)], np.int32))
    fill = aq.paged_batch(2, all_rows.buf, arrays[1].buf, arrays[2].buf, table.shape[1], sum(lens), max(lens), max(lens))
    x = {n: rng.standard_normal((c, h, hd)) for n, c, h in (("k", sum(lens), kv), ("v", sum(lens), kv), ("q", rows, heads))}
    rope = aq.Rope(ctx, hd, THETA)
    got = []
    for st in (dense, strides):
        top = (pages - 1) * st["page_stride"] + (slots - 1) * st["slot_stride"] + (kv - 1) * st["head_stride"] + hd
        k, v = aq.DeviceBuffer(ctx, top * e), aq.DeviceBuffer(ctx, top * e)
        cache = aq.paged_kv(k, v, P.TYPES[cache_t], pages, slots, kv, hd, **st)
        # the rows' stride: past 2^32 bytes for a few rows
        es = P.SIZE[row_t]
        stride = heads * hd if st is dense or rows > 8 else 2 ** 32 // es + 4 * 16
        buf = {n: aq.DeviceBuffer(ctx, ((rows - 1) * stride + heads * hd) * es) for n in ("q", "out")}
        h = {n: aq.heads(b, P.TYPES[row_t], stride, hd) for n, b in buf.items()}
        q = P.store(x["q"], row_t)
        for r in range(rows):
            aq.check(aq.lib().aq_memcpy_htod(ctx.h, C.c_void_p(buf["q"].p.value + r * stride * es), q[r].ctypes.data,
                                             q[r].nbytes))
        kr, vr = P.Rows(ctx, x["k"], row_t), P.Rows(ctx, x["v"], row_t)
        aq.paged_append(ctx, cache, fill, kr.heads_struct(), vr.heads_struct(), rope)
        pos = P.Dev(ctx, np.arange(rows, dtype=np.int32))
        aq.rope_apply(rope, h["q"], h["q"], rows, heads, hd, pos.buf)
        ws = aq.DeviceBuffer(ctx, aq.paged_attention_workspace(ctx, cache, batch, heads))
        aq.paged_attention(ctx, cache, batch, heads, h["q"], h["out"], 0.125, 0, None, ws)
        ctx.sync()
        out = np.zeros_like(q)
        for r in range(rows):
            aq.check(aq.lib().aq_memcpy_dtoh(ctx.h, out[r].ctypes.data, C.c_void_p(buf["out"].p.value + r * stride * es),
                                             out[r].nbytes))
        got.append(P.values(out, row_t))
        for b in (k, v, *buf.values(), ws):
            b.free()
    assert np.all(np.isfinite(got[0])) and np.abs(got[0]).max() > 0.1
    assert np.array_equal(got[0], got[1])


@pytest.mark.parametrize("row_t,cache_t,n_seq,new", [("f32", "bf16", 350, 26), ("bf16", "bf16", 350, 26),
                                                     ("bf16", "bf16", 1100, 9), ("f16", "f16", 1, 36000)])
def test_more_row_tiles_than_one_work_group_divides(ctx, row_t, cache_t, n_seq, new):
    """The plan's own launch: against calls of a few sequences at a time, whose outputs the other tests hold to the
    definition. Two orders of summation: each is within the bound of the same definition."""
    print(f"tiles {row_t}/{cache_t} {n_seq} x {new}", flush=True)
    rng = np.random.default_rng(6)
    lens = [int(n) for n in new + rng.integers(0, 30, n_seq)]
    pg = P.Paged(ctx, rng, [new] * n_seq, lens, 1, 64, 16, cache_t)
    q = P.Rows(ctx, rng.standard_normal((pg.rows, 4, 64)), row_t)
    cache, batch = pg.structs()
    wide = aq.paged_batch(n_seq, pg.dstarts.buf, pg.dlens.buf, pg.dtable.buf, pg.cols, pg.rows, pg.max_rows, 1 << 20)
    step = max(1, n_seq // 11)
    outs = []
    for b in (batch, wide):
        out = P.Rows(ctx, np.full((pg.rows, 4, 64), 9.0), row_t)
        ws = aq.DeviceBuffer(ctx, aq.paged_attention_workspace(ctx, cache, b, 4))
        aq.paged_attention(ctx, cache, b, 4, q.heads_struct(), out.heads_struct(), 0.125, 0, None, ws)
        ctx.sync()
        outs.append(out.get())
    u = 2.0 ** -24
    # values are at most 6 here, and sum |q||k| / 8 over 64 products of mean 0.64 at most 14
    seen = max(lens)
    rel = 2 * 14 * (72 * u + 2.0 ** -21) + (P.HALF_STEP[cache_t] if row_t != "f32" else 2.0 ** -21) + (12 + seen / 4 + 128) * u
    limit = 2 * 6 * rel + 2 * 6 * P.HALF_STEP[row_t]
    for s0 in range(0, n_seq, step):
        s1 = min(s0 + step, n_seq)
        if n_seq == 1:
            check = [(r, min(r + 64, new)) for r in range(0, new, 3000)]
        else:
            check = [(int(pg.starts[s0]), int(pg.starts[s1]))]
        for r0, r1 in check:
            n = s1 - s0
            starts = (pg.starts[s0: s1 + 1] - r0) if n_seq > 1 else np.array([0, r1 - r0], np.int32)
            ln = np.array(lens[s0:s1] if n_seq > 1 else [lens[0] - new + r1], np.int32)
            d = [P.Dev(ctx, a) for a in (starts.astype(np.int32), ln, pg.table[s0:s1])]
            b = aq.paged_batch(n, *(a.buf for a in d), pg.cols, r1 - r0, min(new, r1 - r0), int(ln.max()))
            part, out = P.Rows(ctx, q.values()[r0:r1], row_t), P.Rows(ctx, np.full((r1 - r0, 4, 64), 9.0), row_t)
            ws = aq.DeviceBuffer(ctx, aq.paged_attention_workspace(ctx, cache, b, 4))
            aq.paged_attention(ctx, cache, b, 4, part.heads_struct(), out.heads_struct(), 0.125, 0, None, ws)
            ctx.sync()
            for whole in outs:
                assert np.all(np.isfinite(whole[r0:r1])) and np.all(np.abs(whole[r0:r1] - out.get()) <= limit), (s0, r0)


@pytest.mark.parametrize("row_t,cache_t", PAIRS)
@pytest.mark.parametrize("new", [1, 4, 40])
def test_rows_past_the_bounds_stay(ctx, row_t, cache_t, new):
    """row_start past n_rows, and more rows than max_rows says: rows from n_rows on are not touched, those within both
    are right."""
    print(f"past the bounds {row_t}/{cache_t} new {new}", flush=True)
    rng = np.random.default_rng(7)
    pg = P.Paged(ctx, rng, [new, new, new], [300, 200, 100], 2, 64, 16, cache_t)
    x = rng.standard_normal((pg.rows, 4, 64))
    q, out = P.Rows(ctx, x, row_t), P.Rows(ctx, np.full((pg.rows, 4, 64), 9.0), row_t)
    want, parts = P.attention(pg, q.values(), 0.125)
    limit = P.bound(parts, want, row_t, cache_t, 64)
    cache, _ = pg.structs()
    n = 2 * new + new // 2
    b = aq.paged_batch(3, pg.dstarts.buf, pg.dlens.buf, pg.dtable.buf, pg.cols, n, new, 300)
    ws = aq.DeviceBuffer(ctx, aq.paged_attention_workspace(ctx, cache, b, 4))
    aq.paged_attention(ctx, cache, b, 4, q.heads_struct(), out.heads_struct(), 0.125, 0, None, ws)
    ctx.sync()
    got = out.get()
    assert np.all(got[n:] == 9.0) and np.all(np.abs(got - want)[: 2 * new] <= limit[: 2 * new])


@pytest.mark.parametrize("n_seq", [1, 64, 65, 4096, 5000])
def test_append_of_many_sequences(ctx, n_seq):
    """Each row finds its sequence among thousands, empty ones between them; rows behind the last store nothing."""
    print(f"append of {n_seq} sequences", flush=True)
    rng = np.random.default_rng(n_seq)
    new = [int(n) for n in rng.integers(0, 3, n_seq)]
    new[-1] = 2
    lens = [int(n + x) for n, x in zip(new, rng.integers(0, 9, n_seq))]
    pg = P.Paged(ctx, rng, new, lens, 1, 8, 4, "f32", n_rows=sum(new) + 5)
    k, v = (P.Rows(ctx, rng.standard_normal((pg.rows, 1, 8)), "f32") for _ in range(2))
    want = [pg.k.copy(), pg.v.copy()]
    for s in range(n_seq):
        for i in range(new[s]):
            at = pg.row_of(s, lens[s] - new[s] + i)
            want[0][at], want[1][at] = k.values()[pg.starts[s] + i], v.values()[pg.starts[s] + i]
    cache, batch = pg.structs()
    aq.paged_append(ctx, cache, batch, k.heads_struct(), v.heads_struct())
    ctx.sync()
    for a, b in zip(pg.pools(), want):
        assert np.array_equal(a, b, equal_nan=True)


@pytest.mark.parametrize("row_t,cache_t", PAIRS)
@pytest.mark.parametrize("new", [1, 40])
def test_no_positions_at_all(ctx, row_t, cache_t, new):
    """max_len 0: every row is 0."""
    pg = P.Paged(ctx, np.random.default_rng(1), [new, new], [0, 0], 2, 64, 16, cache_t, max_len=0)
    q, out = (P.Rows(ctx, np.full((pg.rows, 4, 64), x), row_t) for x in (1.0, 9.0))
    cache, batch = pg.structs()
    ws = aq.DeviceBuffer(ctx, aq.paged_attention_workspace(ctx, cache, batch, 4))
    aq.paged_attention(ctx, cache, batch, 4, q.heads_struct(), out.heads_struct(), 0.125, 0, None, ws)
    ctx.sync()
    assert np.all(out.get() == 0.0)
