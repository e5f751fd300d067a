"""Plain forms in 64 bits of the rotary and paged-attention operators, the device arrays of a batch, and the bounds that
the tests hold the kernels to."""
import math

import numpy as np

import aqueduct as aq

TYPES = {"f32": aq.F32, "f16": aq.F16, "bf16": aq.BF16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}
HALF_STEP = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}  # of a value's leading bit, at most
TINY = {"f32": 2.0 ** -149, "f16": 2.0 ** -24, "bf16": 2.0 ** -133}  # the smallest step


def store(x, t):
    """float64 / float32 values as the type's stored array (bf16: uint16, rounded to nearest even)."""
    x = np.asarray(x, np.float32)
    if t == "f32":
        return x.copy()
    if t == "f16":
        return x.astype(np.float16)
    u = np.ascontiguousarray(x).view(np.uint32).astype(np.uint64)
    r = ((u + 0x7FFF + ((u >> 16) & 1)) >> 16).astype(np.uint16)
    return np.where(np.isnan(x), np.uint16(0x7FC0), r)


def values(a, t):
    """The stored array's values, float64."""
    if t == "bf16":
        return (a.astype(np.uint32) << 16).view(np.float32).astype(np.float64)
    return a.astype(np.float64)


STORED = {"f32": np.float32, "f16": np.float16, "bf16": np.uint16}


class Dev:
    """A stored array on the device."""

    def __init__(self, ctx, a):
        self.shape, self.dtype, self.n = a.shape, a.dtype, a.size
        self.buf = aq.DeviceBuffer(ctx, max(a.nbytes, 16))
        if a.size:
            self.buf.upload(a)

    def get(self):
        return self.buf.download(self.dtype, self.n).reshape(self.shape)


class Rows:
    """[rows][heads][head_dim] on the device with `pad` elements between heads and `skip` at the front."""

    def __init__(self, ctx, x, t, pad=0, skip=0, fill=7.0):
        self.t, self.rows, self.heads, self.hd = t, *x.shape
        self.pad, self.skip = pad, skip
        whole = np.full(skip + self.rows * self.heads * (self.hd + pad), fill)
        self.whole = store(whole, t)
        v = self.whole[skip:].reshape(self.rows, self.heads, self.hd + pad)
        v[..., : self.hd] = store(x, t)
        self.dev = Dev(ctx, self.whole)

    def heads_struct(self):
        h = aq.heads(self.dev.buf.p.value + self.skip * SIZE[self.t], TYPES[self.t], self.heads * (self.hd + self.pad),
                     self.hd + self.pad)
        h.keep = self.dev
        return h

    def _view(self, a):
        return a[self.skip:].reshape(self.rows, self.heads, self.hd + self.pad)

    def stored(self):
        return self._view(self.whole)[..., : self.hd]

    def values(self):
        return values(self.stored(), self.t)

    def get(self):
        """The device's rows as values; what lies between them is as it was."""
        a = self.dev.get()
        b, c = a.copy(), self.whole.copy()
        self._view(b)[..., : self.hd] = 0
        self._view(c)[..., : self.hd] = 0
        assert np.array_equal(b.view(np.uint8), c.view(np.uint8)), "written between the rows"
        return values(self._view(a)[..., : self.hd], self.t)


class Paged:
    """A pool of pages and a batch over it. `layout`: "slots" [page][slot][head][dim] or "heads" [page][head][slot][dim].
    Rows past the lengths, and pages nobody owns, hold NaN."""

    def __init__(self, ctx, rng, new, lens, kv, hd, page, t, layout="slots", extra=2, cols=None, order=None,
                 max_rows=None, max_len=None, n_rows=None, sigma=1.0):
        self.ctx, self.new, self.lens, self.kv, self.hd, self.page, self.t = ctx, new, lens, kv, hd, page, t
        self.layout = layout
        need = [-(-max(n, 0) // page) for n in lens]
        n_pages = max(1, sum(need) + extra)
        order = rng.permutation(n_pages) if order is None else order
        self.cols = cols or max(1, max(need, default=0) + 1)
        self.table = np.full((len(lens), self.cols), -1, np.int32)
        at = 0
        for s, n in enumerate(need):
            self.table[s, : min(n, self.cols)] = order[at: at + min(n, self.cols)]
            at += n
        self.starts = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
        self.rows = int(self.starts[-1]) if n_rows is None else n_rows
        self.max_rows = max(new, default=0) if max_rows is None else max_rows
        self.max_len = max(lens, default=0) if max_len is None else max_len
        shape = (n_pages, page, kv, hd)
        self.k, self.v = np.full(shape, np.nan), np.full(shape, np.nan)
        for s, n in enumerate(lens):
            for p in range(0, max(n, 0), page):
                if p // page >= self.cols:
                    break
                m = min(page, n - p)
                self.k[self.table[s, p // page], :m] = rng.standard_normal((m, kv, hd)) * sigma
                self.v[self.table[s, p // page], :m] = rng.standard_normal((m, kv, hd))
        self.upload()

    def _out(self, x):
        a = store(x, self.t)
        return np.ascontiguousarray(a.transpose(0, 2, 1, 3)) if self.layout == "heads" else a

    def upload(self):
        self.k, self.v = values(store(self.k, self.t), self.t), values(store(self.v, self.t), self.t)
        self.dk, self.dv = Dev(self.ctx, self._out(self.k)), Dev(self.ctx, self._out(self.v))
        self.dtable = Dev(self.ctx, self.table)
        self.dstarts, self.dlens = Dev(self.ctx, self.starts), Dev(self.ctx, np.array(self.lens, np.int32))

    def structs(self):
        n, ps, kv, hd = self.k.shape
        if self.layout == "heads":
            st = dict(page_stride=ps * kv * hd, slot_stride=hd, head_stride=ps * hd)
        else:
            st = {}
        cache = aq.paged_kv(self.dk.buf, self.dv.buf, TYPES[self.t], n, ps, kv, hd, **st)
        batch = aq.paged_batch(len(self.lens), self.dstarts.buf, self.dlens.buf, self.dtable.buf, self.cols, self.rows,
                               self.max_rows, self.max_len)
        return cache, batch

    def pools(self):
        """The device's K and V pools as values [page][slot][head][dim]."""
        out = []
        for d in (self.dk, self.dv):
            a = values(d.get(), self.t)
            out.append(a.transpose(0, 2, 1, 3) if self.layout == "heads" else a)
        return out

    def row_of(self, s, p):
        """(page, slot) of a sequence's position, or None."""
        if p < 0 or p // self.page >= self.cols:
            return None
        g = int(self.table[s, p // self.page])
        return (g, p % self.page) if 0 <= g < self.k.shape[0] else None


def attention(pg, q, scale, window=0, gate=None):
    """(outputs, bound) [rows][heads][hd] of the definition in 64 bits: per row the softmax over the positions it sees.
    bound: how far a kernel may be, by arithmetic (see `bound` below), before the output's own rounding."""
    rows, heads, hd = q.shape
    G = heads // pg.kv
    out, mag, top = np.zeros(q.shape), np.zeros(q.shape), np.zeros((rows, heads, 1))
    seen = np.zeros(rows, np.int64)
    for s, (n, length) in enumerate(zip(pg.new, pg.lens)):
        for i in range(n):
            r, pos = int(pg.starts[s]) + i, length - n + i
            if r >= rows:
                continue
            lo = max(0, pos + 1 - window) if window else 0
            places = [pg.row_of(s, p) for p in range(lo, min(pos + 1, pg.max_len))]
            places = np.array([x for x in places if x is not None], np.int64).reshape(-1, 2)
            seen[r] = len(places)
            if not len(places):
                continue
            k, v = pg.k[places[:, 0], places[:, 1]], pg.v[places[:, 0], places[:, 1]]
            for h in range(heads):
                x = k[:, h // G] @ q[r, h] * scale
                with np.errstate(invalid="ignore", over="ignore"):
                    p = np.exp(x - x.max())
                    p /= p.sum()
                    vv = v[:, h // G]
                    out[r, h] = (p[:, None] * vv).sum(0)
                    mag[r, h] = (p[:, None] * np.abs(vv)).sum(0)
                    top[r, h] = (np.abs(k[:, h // G]) @ np.abs(q[r, h])).max() * scale
    if gate is not None:
        g = 1.0 / (1.0 + np.exp(-gate))
        out, mag = out * g, mag * g
    return out, (mag, top, seen)


def bound(parts, want, row_t, cache_t, hd):
    """Largest error of an output by the rounding of each step (u = 2^-24 a 32-bit rounding):
    scores: a sum of hd products in 32 bits, in any order: hd u T, T the largest sum of |q||k| scale; queries in pieces
      (f32 rows over f16: two f16 pieces, 2^-22; over bf16 three, 2^-24): 2^-21 T; the scale's and exponent's
      factors and their fused rounding: 8 u T
    probabilities: exp2's error 4 u, their rounding to the cache's type where the rows have it (half a step), else to
      2^-21 in pieces; a score's error d moves a probability by a factor of 1 + d, and their sum as much
    sums: the probabilities' sum and the outputs over the positions in 32 bits, rescaled at most once a tile: each adds
      at most (positions / 8 + 64) u to an output's magnitude (sums of 8 or 32 positions inside an instruction)
    all of that times sum p |v|; then the gate (8 u) and the output's rounding."""
    mag, top, seen = parts
    u = 2.0 ** -24
    d = top * ((hd + 8) * u + 2.0 ** -21)
    p = HALF_STEP[cache_t] if row_t != "f32" else 2.0 ** -21
    rel = 2 * d + p + (4 + 8 + 2 * (seen[:, None, None] / 8 + 64)) * u
    return 1.05 * mag * rel + np.abs(want) * HALF_STEP[row_t] + TINY[row_t]


def frequencies(dim, theta, scaling="none", factor=1.0, orig=0, fast=32.0, slow=1.0):
    i = np.arange(dim // 2, dtype=np.float64)
    theta = float(np.float32(theta))
    f = theta ** (-2.0 * i / dim)
    if scaling == "linear":
        return f / factor, 1.0
    if scaling == "yarn":
        def at(turns):
            return dim * math.log(orig / (turns * 2 * math.pi)) / (2 * math.log(theta))
        lo, hi = max(math.floor(at(fast)), 0), min(math.ceil(at(slow)), dim - 1)
        slowed = np.clip((i - lo) / max(hi - lo, 1e-3), 0, 1)
        return f / factor * slowed + f * (1 - slowed), 0.1 * math.log(factor) + 1 if factor > 1 else 1.0
    return f, 1.0


def rotate(x, pos, dim, layout, freq, gain=1.0, inverse=False):
    """x [rows][heads][hd] turned by pos (float64)."""
    a = np.asarray(pos, np.float64)[:, None, None] * freq
    c, s = np.cos(a) * gain, np.sin(a) * gain * (-1 if inverse else 1)
    y = x.copy()
    i, j = (slice(0, dim // 2), slice(dim // 2, dim)) if layout == "half" else (slice(0, dim, 2), slice(1, dim, 2))
    y[..., i], y[..., j] = x[..., i] * c - x[..., j] * s, x[..., j] * c + x[..., i] * s
    return y


def rotate_bound(x, want, t, gain=1.0):
    """The angle is right to 2^-24 of a turn and the sine to 4 u, so a pair (a, b) moves by at most (2 pi + 8) u |(a, b)|
    gain, plus three 32-bit roundings; |(a, b)| is at most sqrt(2) of the head's largest value. Then the output's
    rounding."""
    big = np.abs(x).max(-1, keepdims=True) * math.sqrt(2) * gain
    return big * 20 * 2.0 ** -24 + np.abs(want) * HALF_STEP[t] + TINY[t]
