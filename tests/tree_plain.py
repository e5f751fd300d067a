"""Plain forms in 64 bits of the head norms with the rotation, tree attention, accepted paths and page tables, and the bounds
that the tests hold the kernels to (paged_plain.py has those that they share with the rotary and paged operators)."""
import numpy as np

import paged_plain as P

U = 2.0 ** -24


def normed(x, w, eps):
    return x / np.sqrt((x ** 2).mean(-1, keepdims=True) + eps) * w


def norm_bound(x, w, eps, want, t, rotated=0, gain=1.0):
    """The sum of hd squares in 32 bits, in any order, is off by hd u of itself, the mean and eps by 2 u, of which the root
    takes half; the reciprocal root 4 u, the two products 2 u: (hd / 2 + 7) u of each normed value. A turned pair moves by
    sqrt(2) of its larger value's error at most, and by the rotation's own (paged_plain.rotate_bound, which has the output's
    rounding)."""
    y = normed(x, w, eps)
    rel = (x.shape[-1] / 2 + 7) * U * 1.05
    small = np.abs(y) * rel + np.abs(want) * P.HALF_STEP[t] + P.TINY[t]
    big = np.abs(y).max(-1, keepdims=True) * 1.4143 * gain * rel + P.rotate_bound(y, want, t, gain)
    return np.where(np.arange(x.shape[-1]) < rotated, big, small)


def pack(masks, words):
    """Truth values [rows][new rows] as mask words [rows][words]."""
    out = np.zeros((len(masks), words * 32), np.uint8)
    for r, m in enumerate(masks):
        out[r, : len(m)] = m
    return np.packbits(out, axis=1, bitorder="little").view(np.uint32)


def random_trees(rng, new, near=4.0):
    """For each sequence's new rows their masks: each row hangs on an earlier one, mostly a near one."""
    rows = []
    for n in new:
        own = np.zeros((n, n), bool)
        for i in range(n):
            if i:
                own[i] = own[max(0, i - 1 - int(rng.exponential(near)))]
            own[i, i] = True
        rows += list(own)
    return rows


def tree_attention(pg, masks, q, scale, window=0, gate=None):
    """(outputs, what paged_plain.bound takes) of the definition in 64 bits: per row the softmax over what stands before its
    sequence's new rows (with a window, the last window - n of it, for a mask of n bits) and the new rows of its mask."""
    rows, heads, hd = q.shape
    G = heads // pg.kv
    out, mag, top = np.zeros(q.shape), np.zeros(q.shape), np.zeros((rows, heads, 1))
    seen = np.zeros(rows, np.int64)
    for s, (n, length) in enumerate(zip(pg.new, pg.lens)):
        base = max(length, 0) - n
        for i in range(n):
            r = int(pg.starts[s]) + i
            if r >= rows:
                continue
            m = masks[r]
            lo = max(0, min(base, base + int(np.sum(m)) - window)) if window else 0
            at = list(range(lo, base)) + [base + j for j in range(n) if j < len(m) and m[j]]
            places = [pg.row_of(s, p) for p in at if p < pg.max_len]
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


class Tables:
    """The page tables of a pool as the device keeps them, and a step over them by its definition, a request at a time."""

    def __init__(self, n_seq, max_pages, n_pages, page):
        self.n_seq, self.max_pages, self.n_pages, self.page = n_seq, max_pages, n_pages, page
        self.pages = np.full((n_seq, max_pages), -7, np.int32)
        self.held = np.zeros(n_seq, np.int32)
        self.ring = np.arange(n_pages, dtype=np.int32)
        self.first, self.count = 0, n_pages

    def step(self, before, new, n_rows, depth=None):
        """What a step writes: (row_start, kv_len, missing, pos, slots); the tables afterwards are in self."""
        free, first, used, back, short = self.count, self.first, 0, 0, False
        start, length, missing = [0], [], []
        pos, slots = np.zeros(n_rows, np.int32), np.full(n_rows, -1, np.int64)
        old, old_held = self.pages.copy(), self.held.copy()
        for s in range(self.n_seq):
            b, n = max(int(before[s]), 0), int(new[s])
            total = 0 if n < 0 else b + n
            need = -(-total // self.page)
            want, have = min(need, self.max_pages), int(old_held[s])
            length.append(total)
            missing.append(need - want)
            if want > have:
                short = short or used + want - have > free
                for c in range(have, want):
                    self.pages[s, c] = -1 if short else self.ring[(first + used + c - have) % self.n_pages]
                if short:
                    missing[-1] += want - have
                else:
                    used += want - have
                    self.held[s] = want
            else:
                for c in range(want, have):
                    self.ring[(first + free + back) % self.n_pages] = old[s, c]
                    back += 1
                self.held[s] = want
            for i in range(max(n, 0)):
                r = start[-1] + i
                if r >= n_rows:
                    break
                p = b + i
                pos[r] = p if depth is None else b + depth[r]
                if p // self.page < want and 0 <= self.pages[s, p // self.page] < self.n_pages:
                    slots[r] = int(self.pages[s, p // self.page]) * self.page + p % self.page
            start.append(start[-1] + max(n, 0))
        self.first, self.count = (first + used) % self.n_pages, free - used + back
        return (np.array(start, np.int32), np.array(length, np.int32), np.array(missing, np.int32), pos, slots)
