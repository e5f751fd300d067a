"""What the rotary and paged-attention calls refuse, with their codes and texts: every refusal comes before anything
touches a device, so a context that names a device, and addresses that are never read, are enough (no GPU needed)."""
import ctypes as C

import pytest

import aqueduct as aq

FAKE = 0x10000  # an address: 16-byte aligned, never dereferenced by a refused call


class FakeCtx:
    """An aq_ctx's first field (the device) and zeros: for calls that are refused before they use it."""

    def __init__(self):
        self.mem = C.create_string_buffer(256)
        self.h = C.c_void_p(C.addressof(self.mem))


class FakeRope:
    """An aq_rope: context pointer, dim, layout, then zeros."""

    def __init__(self, ctx, dim, layout=0):
        self.ctx, self.mem = ctx, C.create_string_buffer(256)
        C.c_void_p.from_buffer(self.mem, 0).value = ctx.h.value
        C.c_uint32.from_buffer(self.mem, 8).value = dim
        C.c_uint32.from_buffer(self.mem, 12).value = layout
        self.h = C.c_void_p(C.addressof(self.mem))


@pytest.fixture()
def ctx():
    return FakeCtx()


def good_kv(**kw):
    a = dict(k=FAKE, v=FAKE, type=aq.F16, n_pages=64, page_size=16, n_head_kv=2, head_dim=64)
    a.update(kw)
    return aq.paged_kv(**a)


def good_batch(**kw):
    a = dict(n_seq=2, row_start=FAKE, kv_len=FAKE, pages=FAKE, max_pages=8, n_rows=4, max_rows=2, max_len=100)
    a.update(kw)
    return aq.paged_batch(**a)


def rows(t=aq.F16, heads=2, hd=64, data=FAKE, row=None, head=None):
    return aq.heads(data, t, heads * hd if row is None else row, hd if head is None else head)


def refused(code, text, call, *args, **kw):
    with pytest.raises(aq.AqError) as e:
        call(*args, **kw)
    assert e.value.code == code and text in str(e.value), str(e.value)


@pytest.mark.parametrize("kw,text", [
    (dict(dim=0), "dim"), (dict(dim=7), "dim"), (dict(dim=64, theta=0.5), "theta"),
    (dict(dim=64, theta=float("nan")), "theta"), (dict(dim=64, scaling="linear", factor=0.0), "factor"),
    (dict(dim=64, scaling="yarn", factor=4.0), "orig_ctx"), (dict(dim=64, theta=1.0, scaling="yarn", factor=4.0, orig_ctx=9), "theta > 1"),
    (dict(dim=64, scaling="yarn", factor=4.0, orig_ctx=9, beta_fast=1.0, beta_slow=2.0), "beta"),
    (dict(dim=64, scaling="yarn", factor=4.0, orig_ctx=9, attn_factor=-1.0), "attn_factor"),
    (dict(dim=64, layout="other"), "layout"), (dict(dim=64, scaling="other"), "scaling")])
def test_rope_settings(ctx, kw, text):
    refused(aq.AQ_EINVAL, text, aq.Rope, ctx, **kw)


def test_rope_apply(ctx):
    rope, x = FakeRope(ctx, 64), rows()

    def go(code, text, x=x, y=None, n=3, heads=2, hd=64, pos=FAKE, r=rope):
        refused(code, text, aq.rope_apply, r, x, y or rows(data=2 * FAKE), n, heads, hd, pos)

    go(aq.AQ_EINVAL, "rotated", hd=32)
    go(aq.AQ_EINVAL, "type", x=rows(t=aq.Q4_K))
    go(aq.AQ_EINVAL, "different types", y=rows(t=aq.BF16, data=2 * FAKE))
    go(aq.AQ_EINVAL, "null", x=rows(data=None))
    go(aq.AQ_EINVAL, "aligned", x=rows(data=FAKE + 1))
    go(aq.AQ_EINVAL, "rows overlap", x=rows(row=32))
    go(aq.AQ_EINVAL, "heads overlap", x=rows(head=63))
    go(aq.AQ_EINVAL, "strides", x=rows(row=-128))
    go(aq.AQ_EINVAL, "same strides", y=rows(row=256))
    go(aq.AQ_EINVAL, "pos_dev", pos=None)
    go(aq.AQ_EINVAL, "size", n=1 << 24)
    go(aq.AQ_EINVAL, "odd", hd=65, x=rows(hd=65), y=rows(hd=65, data=2 * FAKE), r=FakeRope(ctx, 64, 1))
    aq.rope_apply(rope, x, rows(), 0, 2, 64, FAKE)  # nothing to do
    assert aq.lib().aq_rope_apply(None, None, None, 0, 0, 0, None, 0, None) == aq.AQ_EINVAL


BAD_CACHES = [
    (aq.AQ_EINVAL, "cache type", dict(type=aq.Q8_0)), (aq.AQ_EINVAL, "pages", dict(n_pages=0)),
    (aq.AQ_EINVAL, "pages", dict(page_size=0)), (aq.AQ_EINVAL, "null", dict(k=None)), (aq.AQ_EINVAL, "null", dict(v=None)),
    (aq.AQ_EINVAL, "n_head_kv", dict(n_head_kv=0)), (aq.AQ_EUNSUP, "head_dim", dict(head_dim=60)),
    (aq.AQ_EUNSUP, "head_dim", dict(head_dim=264)), (aq.AQ_EUNSUP, "head_dim", dict(head_dim=0)),
    (aq.AQ_EINVAL, "16-byte", dict(k=FAKE + 8)), (aq.AQ_EINVAL, "16 bytes", dict(slot_stride=132)),
    (aq.AQ_EINVAL, "heads of a page", dict(head_stride=56)), (aq.AQ_EINVAL, "slots of a page", dict(slot_stride=56)),
    (aq.AQ_EINVAL, "pages overlap", dict(page_stride=0)), (aq.AQ_EINVAL, "strides", dict(page_stride=-2048)),
    (aq.AQ_EUNSUP, "2^32 units", dict(n_pages=1 << 30, page_stride=(1 << 30) + 8)),
]
BAD_BATCHES = [
    ("null batch", dict(row_start=None)), ("null batch", dict(kv_len=None)), ("null batch", dict(pages=None)),
    ("max_pages", dict(max_pages=0)), ("batch size", dict(n_rows=1 << 24)), ("batch size", dict(n_seq=1 << 24)),
    ("2^31 positions", dict(max_pages=1 << 27)),
]


def calls(ctx):
    def append(kv, b):
        aq.paged_append(ctx, kv, b, rows(), rows())

    def attend(kv, b):
        aq.paged_attention(ctx, kv, b, 4, rows(heads=4), rows(heads=4, data=2 * FAKE), 0.1, workspace=FAKE,
                           workspace_bytes=1 << 40)

    def size(kv, b):
        aq.paged_attention_workspace(ctx, kv, b, 4)

    return append, attend, size


@pytest.mark.parametrize("which", [0, 1, 2])
@pytest.mark.parametrize("code,text,kw", BAD_CACHES)
def test_caches(ctx, which, code, text, kw):
    refused(code, text, calls(ctx)[which], good_kv(**kw), good_batch())


@pytest.mark.parametrize("which", [0, 1, 2])
@pytest.mark.parametrize("text,kw", BAD_BATCHES)
def test_batches(ctx, which, text, kw):
    refused(aq.AQ_EINVAL, text, calls(ctx)[which], good_kv(), good_batch(**kw))


def test_append(ctx):
    def go(text, k=rows(), v=rows(), kv=good_kv(), code=aq.AQ_EINVAL, **kw):
        refused(code, text, aq.paged_append, ctx, kv, good_batch(), k, v, **kw)

    rope = FakeRope(ctx, 64)
    go("k: null", k=None)
    go("v: null", v=rows(data=None))
    go("different types", v=rows(t=aq.F32))
    go("of the cache's type", k=rows(t=aq.BF16), v=rows(t=aq.BF16))
    go("of the cache's type", k=rows(), v=rows(), kv=good_kv(type=aq.F32))
    go("q without a rope", q=rows(), q_out=rows(), n_head=2)
    go("go together", rope=rope, q=rows(), n_head=2)
    go("n_head", rope=rope, q=rows(), q_out=rows(), n_head=0)
    go("different types", rope=rope, q=rows(t=aq.F32), q_out=rows(t=aq.F32), n_head=2)
    go("same strides", rope=rope, q=rows(), q_out=rows(row=256), n_head=2)
    go("rotated", rope=FakeRope(ctx, 66))
    other = FakeCtx()
    C.c_int.from_buffer(other.mem, 0).value = 1
    go("another device", rope=FakeRope(other, 64))
    aq.paged_append(ctx, good_kv(), good_batch(n_rows=0), rows(), rows())  # nothing to do
    aq.paged_append(ctx, good_kv(), good_batch(n_seq=0), rows(), rows())
    assert aq.lib().aq_paged_append(None, *[None] * 7, 0, None) == aq.AQ_EINVAL


def test_attention(ctx):
    def go(text, q=rows(heads=4), out=rows(heads=4, data=2 * FAKE), kv=good_kv(), heads=4, scale=0.1, gate=None,
           ws=FAKE, size=1 << 40, code=aq.AQ_EINVAL, batch=None):
        refused(code, text, aq.paged_attention, ctx, kv, batch or good_batch(), heads, q, out, scale, 0, gate, ws, size)

    go("n_head", heads=3)
    go("n_head", heads=0)
    go("q: null", q=None)
    go("out: null", out=rows(heads=4, data=None))
    go("gate: type", gate=rows(t=2))
    go("of the cache's type", q=rows(t=aq.BF16, heads=4), out=rows(t=aq.BF16, heads=4))
    go("different types", out=rows(t=aq.F32, heads=4))
    go("different types", gate=rows(t=aq.F32, heads=4))
    for scale in (0.0, -1.0, float("inf"), float("nan")):
        go("scale", scale=scale)
    go("workspace", ws=None)
    go("workspace", ws=FAKE + 4)
    need = aq.paged_attention_workspace(ctx, good_kv(), good_batch(), 4)
    assert need > 0
    go(f"{need} needed", size=need - 1)
    go("2^31 units", batch=good_batch(n_seq=1 << 23, n_rows=1 << 23, max_pages=1 << 23, max_len=(1 << 27) - 1),
       code=aq.AQ_EUNSUP)
    aq.paged_attention(ctx, good_kv(), good_batch(n_rows=0), 4, rows(heads=4), rows(heads=4), 0.1)  # nothing to do
    assert aq.lib().aq_paged_attention(None, *[None] * 2, 4, None, None, 0.1, 0, None, None, 0, None) == aq.AQ_EINVAL
    assert aq.lib().aq_paged_attention_workspace(ctx.h, C.byref(good_kv()), C.byref(good_batch()), 4, None) == aq.AQ_EINVAL


def test_empty_batches_need_no_rows(ctx):
    """Row tensors without rows may have no address."""
    none, batch = rows(data=None), good_batch(n_rows=0)
    aq.paged_append(ctx, good_kv(), batch, none, none)
    aq.paged_append(ctx, good_kv(), batch, none, none, FakeRope(ctx, 64), none, none, 2)
    aq.paged_attention(ctx, good_kv(), batch, 2, none, none, 0.1, 0, none)
    aq.rope_apply(FakeRope(ctx, 64), none, none, 0, 2, 64, None)


def test_reach_of_a_table(ctx):
    """Up to 2^31 - 1024 positions; heads any distance apart."""
    most = ((1 << 31) - 1024) // 16
    assert aq.paged_attention_workspace(ctx, good_kv(), good_batch(max_pages=most), 4) > 0
    refused(aq.AQ_EINVAL, "2^31 positions", aq.paged_attention_workspace, ctx, good_kv(), good_batch(max_pages=most + 1), 4)
    assert aq.paged_attention_workspace(ctx, good_kv(head_stride=1 << 39), good_batch(), 4) > 0


def test_rows_of_a_kv_head(ctx):
    """Rows times the query heads of a K/V head stay 1024 under 2^31."""
    kv, most = good_kv(n_head_kv=1), ((1 << 31) - 1024) // 256
    assert aq.paged_attention_workspace(ctx, kv, good_batch(n_rows=most, max_len=16), 256) > 0
    refused(aq.AQ_EINVAL, "batch size", aq.paged_attention_workspace, ctx, kv, good_batch(n_rows=most + 1, max_len=16), 256)


def test_workspace_of_larger_bounds_serves_smaller_batches(ctx):
    """A workspace made for a batch's largest bounds is enough for every batch within them."""
    import random
    rng = random.Random(1)

    def need(n_seq, per_seq, max_len, kv, heads):
        batch = good_batch(n_seq=n_seq, n_rows=n_seq * per_seq, max_rows=per_seq, max_pages=1 << 12, max_len=max_len)
        return aq.paged_attention_workspace(ctx, kv, batch, heads)

    def log(lo, hi):
        return int(round(lo * (hi / lo) ** rng.random()))

    for _ in range(4000):
        n_kv = rng.choice([1, 2, 4, 8])
        kv = good_kv(n_head_kv=n_kv, head_dim=rng.choice([64, 80, 128, 192, 256]), type=rng.choice([aq.F32, aq.F16, aq.BF16]))
        heads = n_kv * rng.choice([1, 2, 4, 6, 12])
        n_seq = log(1, 3000)
        big = [n_seq, log(1, max(30000 // n_seq, 1)), log(1, 60000)]
        small = [log(1, b) for b in big]
        assert need(*small, kv, heads) <= need(*big, kv, heads), (small, big, kv.type, kv.head_dim, n_kv, heads)


def test_attention_in_place(ctx):
    """The output over the queries or the gate has their strides, where those matter."""
    def go(text, q, out, gate=None, heads=4, **kw):
        refused(aq.AQ_EINVAL, text, aq.paged_attention, ctx, good_kv(), good_batch(**kw), heads, q, out, 0.1, 0, gate, FAKE, 0)

    def at(place, **kw):
        return rows(heads=4, data=place, **kw)

    go("same strides", at(FAKE), at(FAKE, row=512))
    go("same strides", at(FAKE, head=128, row=512), at(FAKE, row=512))
    go("same strides", at(2 * FAKE), at(FAKE), at(FAKE, row=512))
    go("needed", at(FAKE), at(FAKE))  # no workspace: everything before that is as it should be
    go("needed", at(2 * FAKE), at(FAKE), at(FAKE))
    go("needed", at(FAKE), at(FAKE, row=512), n_rows=1)
    go("needed", at(FAKE), at(2 * FAKE, row=512))
