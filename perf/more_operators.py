"""A step of a served batch with trees of drafted tokens over a paged K/V cache, as cases that can be timed: page tables and
slot maps from the requests' lengths, queries and keys normed head by head with the rotation in the same pass, attention of
the trees, and the accepted paths kept.

A case is a dict of plain values; its "kind" says which operator it runs:

  norm    q and k rows: each head's root mean square norm and its rotation, in one pass
  append  the same on the way into the pages, with the values
  tables  pages for what grows, pages back from what shrank or ended, the new rows' starts, positions and slots
  tree    a tree of drafted tokens for each sequence over its pages: every row sees what came before and its own ancestors
  commit  the K/V rows of each accepted path moved behind the sequence, in every layer's pages

`own` false: elementary torch operations in 32 bits (angles in 64), rounded once at the end. `own` true: the calls of the
`aqueduct` package, queued on the one stream that a program keeps.
"""
import math
import os
import sys

import numpy as np
import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
ROW_BYTES = {"f32": 4, "f16": 2, "bf16": 2}
THETA, EPS = 1e7, 1e-6
GOLDEN = 0.6180339887498949


# ------------------------------------------------------------------------------------------------------- cases
def norm(rows, heads, kv, head_dim, dim, layout, dtype, first=0):
    return {"kind": "norm", "rows": rows, "heads": heads, "kv": kv, "head_dim": head_dim, "dim": dim, "layout": layout,
            "dtype": dtype, "first": first}


def append(seqs, new, context, heads, kv, head_dim, dim, layout, page, dtype, cache):
    return {"kind": "append", "seqs": seqs, "new": new, "context": context, "heads": heads, "kv": kv,
            "head_dim": head_dim, "dim": dim, "layout": layout, "page": page, "dtype": dtype, "cache": cache}


def tables(seqs, new, context, page, ended, spare):
    """`ended`: the share of requests that end with this step; `spare`: the free pages, as a share of what the step takes."""
    return {"kind": "tables", "seqs": seqs, "new": new, "context": context, "page": page, "ended": ended, "spare": spare}


def tree(seqs, new, context, heads, kv, head_dim, page, dtype, cache, window=0, gate=False):
    return {"kind": "tree", "seqs": seqs, "new": new, "context": context, "heads": heads, "kv": kv,
            "head_dim": head_dim, "page": page, "dtype": dtype, "cache": cache, "window": window, "gate": gate}


def commit(seqs, new, accepted, context, layers, kv, head_dim, page, cache):
    return {"kind": "commit", "seqs": seqs, "new": new, "accepted": accepted, "context": context, "layers": layers,
            "kv": kv, "head_dim": head_dim, "page": page, "cache": cache}


def listed():
    return [
        # one token's query and key heads of the 27B shapes, a quarter of each head rotated: launch and latency
        dict(norm(1, 24, 4, 256, 64, "half", "f32", first=4097), name="norm_f32_1x28x256"),
        # a whole prompt's heads, rotated in full
        dict(norm(8191, 32, 8, 128, 128, "half", "bf16", first=60001), name="norm_bf16_8191x40x128"),
        # a decode step of a served batch: a token for each of 48 sequences
        dict(append(48, 1, 4000, 32, 8, 128, 128, "half", 16, "bf16", "bf16"), name="append_norm_bf16_48x1"),
        # ragged prompt chunks of four requests, f32 activations into a 16-bit cache
        dict(append(4, 1500, 900, 24, 4, 256, 64, "interleaved", 64, "f32", "f16"), name="append_norm_f32_f16_4x1500"),
        # the tables of a decode step of 48 requests, a few of which have just ended
        dict(tables(48, 1, 4000, 16, 0.05, 1.5), name="tables_48x1"),
        # the tables of a large batch that takes up prompts: more pages asked for than are free
        dict(tables(700, 90, 2000, 16, 0.2, 0.9), name="tables_700x90"),
        # a small model's tree of a few drafts: launch and latency
        dict(tree(1, 8, 300, 4, 2, 64, 16, "f32", "f32"), name="tree_f32_1x8_at_300"),
        # a tree of 26 drafts in the 27B's heads, f32 rows over half as much cache, its output gate
        dict(tree(1, 26, 8000, 24, 4, 256, 64, "f32", "f16", gate=True), name="tree_f32_f16_1x26_at_8000"),
        # a served batch's trees
        dict(tree(16, 32, 3000, 32, 8, 128, 16, "bf16", "bf16"), name="tree_bf16_16x32_at_3000"),
        # large trees over long contexts
        dict(tree(4, 64, 16000, 24, 4, 256, 32, "bf16", "bf16", gate=True), name="tree_bf16_4x64_at_16000"),
        # one conversation's accepted path, the 16 attention layers of the 27B shapes
        dict(commit(1, 26, 5, 2000, 16, 4, 256, 64, "f16"), name="commit_f16_1x5_16"),
        # a served batch's accepted paths
        dict(commit(48, 32, 8, 100, 16, 8, 128, 16, "bf16"), name="commit_bf16_48x8_16"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _draw_heads(rng):
    return rng.choice([(24, 4, 256), (24, 4, 256), (32, 8, 128), (28, 4, 128), (4, 2, 64), (16, 16, 64), (14, 2, 64),
                       (8, 1, 128), (16, 16, 80), (20, 4, 96), (16, 4, 192)])


def _draw_types(rng):
    return rng.choice([("f16", "f16"), ("bf16", "bf16"), ("f32", "f32"), ("f32", "f16"), ("f32", "bf16")])


def draw(rng):
    kind = rng.choice(["norm", "append", "tables", "tree", "tree", "tree", "commit"])
    page = rng.choice([16, 16, 32, 64, 128, 24])
    layout = rng.choice(["half", "half", "interleaved"])
    heads, kv, hd = _draw_heads(rng)
    dim = rng.choice([hd, hd // 2, 32])
    dtype, cache = _draw_types(rng)
    if kind == "norm":
        return norm(_log_int(rng, 1, 7000), heads, kv, hd, dim, layout, rng.choice(["f32", "f16", "bf16"]),
                    _log_int(rng, 1, 200000))
    if kind == "append":
        seqs = _log_int(rng, 1, 64)
        return append(seqs, _log_int(rng, 1, max(2, 6000 // seqs)), _log_int(rng, 1, 4000), heads, kv, hd, dim, layout,
                      page, dtype, cache)
    if kind == "tables":
        seqs = _log_int(rng, 1, 1500)
        return tables(seqs, _log_int(rng, 1, max(2, 60000 // seqs)), _log_int(rng, 1, 4000), page,
                      rng.choice([0.0, 0.05, 0.3]), rng.choice([0.5, 0.95, 1.1, 3.0]))
    if kind == "commit":
        seqs, layers = _log_int(rng, 1, 48), rng.choice([1, 2, 16, 24])
        new = rng.randint(8, 64)
        return commit(seqs, new, rng.randint(1, min(new // 2, 12)), rng.randint(1, max(2, 6000 // (seqs * layers))),
                      layers, kv, hd, page, cache)
    seqs, new = _log_int(rng, 1, 32), _log_int(rng, 2, 130)
    most = 250_000_000 // (seqs * new * heads * (8 if dtype == "f32" else 1))
    context = _log_int(rng, 1, max(2, min(16000, most, 170_000_000 // (seqs * kv * hd))))
    return tree(seqs, new, context, heads, kv, hd, page, dtype, cache, rng.choice([0, 0, 0, _log_int(rng, 16, 4096)]),
                rng.random() < 0.3)


def _ragged(mean, n, shift):
    """n whole numbers spread between a quarter and seven quarters of `mean`; one alone, or a mean of 1, is `mean`."""
    if n == 1 or mean <= 1:
        return [mean] * n
    return [max(1, int(mean * (0.25 + 1.5 * ((i * GOLDEN + shift) % 1.0)))) for i in range(n)]


def _lengths(case):
    """Each sequence's new rows, and its length with them."""
    new = _ragged(case["new"], case["seqs"], 0.5)
    before = _ragged(case["context"], case["seqs"], 0.25)
    return new, [a + b for a, b in zip(new, before)]


def _requests(case):
    """The tables' requests: positions held before, new rows (-1: ended), pages held, and the pool's free pages and size."""
    page = case["page"]
    new, lens = _lengths(case)
    before = [n - m for n, m in zip(lens, new)]
    ended = [(i * GOLDEN + 0.1) % 1.0 < case["ended"] for i in range(case["seqs"])]
    fresh = [(i * GOLDEN + 0.7) % 1.0 < 0.1 for i in range(case["seqs"])]  # requests that begin: nothing before
    before = [0 if f else b for f, b in zip(fresh, before)]
    # some hold a page more than their length needs: drafts that were not accepted reached into it
    held = [-(-b // page) + (1 if b and (i * GOLDEN) % 1.0 < 0.15 else 0) for i, b in enumerate(before)]
    new = [-1 if e and not f else n for e, f, n in zip(ended, fresh, new)]
    want = [0 if n < 0 else -(-(b + n) // page) for b, n in zip(before, new)]
    takes = sum(max(0, w - h) for w, h in zip(want, held))
    free = int(takes * case["spare"])
    return before, new, held, want, free, sum(held) + free + 5


# ------------------------------------------------------------------------------------------------------ prepare
def _normal(g, shape, dtype, sigma=1.0):
    return (torch.randn(shape, generator=g, device="cuda") * sigma).to(dtype)


def _ints(values, dtype=torch.int32):
    return torch.tensor(values, dtype=dtype, device="cuda")


def _weights(g, head_dim):
    """Each head's norm weights: near one, as trained ones are."""
    return 1.0 + 0.2 * torch.randn(head_dim, generator=g, device="cuda")


def _prepare_norm(case, g):
    dt, hd = DTYPES[case["dtype"]], case["head_dim"]
    jump = int(torch.randint(0, 4096, (1,), generator=g, device="cuda"))
    q = _normal(g, (case["rows"], case["heads"], hd), dt, 2.5)
    k = _normal(g, (case["rows"], case["kv"], hd), dt, 4.0)
    return {"q": q, "k": k, "q_weight": _weights(g, hd), "k_weight": _weights(g, hd), "q_out": torch.zeros_like(q),
            "k_out": torch.zeros_like(k),
            "pos": torch.arange(case["rows"], device="cuda", dtype=torch.int32) + (case["first"] + jump)}


def _prepare_pages(case, g, layers=0):
    new, lens = _lengths(case)
    page, ct = case["page"], DTYPES[case["cache"]]
    need = [-(-n // page) for n in lens]
    n_pages, cols = sum(need) + 3, max(need) + 1
    order = torch.randperm(n_pages, generator=g, device="cuda").to(torch.int32).cpu()
    table, at = torch.full((case["seqs"], cols), -1, dtype=torch.int32), 0
    for s, n in enumerate(need):
        table[s, :n] = order[at:at + n]
        at += n
    starts = [sum(new[:s]) for s in range(case["seqs"] + 1)]
    shape = (n_pages, page, case["kv"], case["head_dim"])
    shape = (layers, *shape) if layers else shape
    return {"k": _normal(g, shape, ct), "v": _normal(g, shape, ct), "table": table.cuda(), "starts": _ints(starts),
            "lens": _ints(lens), "rows": starts[-1], "most_new": max(new), "longest": max(lens)}


def _prepare_append(case, g):
    s, dt, hd = _prepare_pages(case, g), DTYPES[case["dtype"]], case["head_dim"]
    s["q"] = _normal(g, (s["rows"], case["heads"], hd), dt, 2.5)
    s["new_k"] = _normal(g, (s["rows"], case["kv"], hd), dt, 4.0)
    s["new_v"] = _normal(g, (s["rows"], case["kv"], hd), dt)
    s["q_weight"], s["k_weight"] = _weights(g, hd), _weights(g, hd)
    s["q_out"] = torch.zeros_like(s["q"])
    return s


def _prepare_tables(case, g):
    before, new, held, want, free, n_pages = _requests(case)
    cols = max(max(held), max(want)) + 1
    order = torch.randperm(n_pages, generator=g, device="cuda").to(torch.int32).cpu()
    pages, at = torch.full((case["seqs"], cols), -1, dtype=torch.int32), 0
    for s, n in enumerate(held):
        pages[s, :n] = order[at:at + n]
        at += n
    first = int(torch.randint(0, n_pages, (1,), generator=g, device="cuda"))  # the ring begins anywhere
    ring = torch.full((n_pages,), -1, dtype=torch.int32)
    ring[(first + torch.arange(free)) % n_pages] = order[at:at + free]
    n, rows = case["seqs"], sum(max(m, 0) for m in new)
    return {"pages": pages.cuda(), "held": _ints(held), "ring": ring.cuda(), "state": _ints([first, free, 0, 0]),
            "before": _ints(before), "new": _ints(new), "rows": rows,
            "held_out": _ints([0] * n), "state_out": _ints([0] * 4), "starts": _ints([0] * (n + 1)),
            "lens": _ints([0] * n), "missing": _ints([0] * n), "pos": _ints([0] * rows),
            "slots": _ints([0] * rows, torch.int64)}


def _draft_trees(new, rng):
    """Mask words [rows][words] of one random tree a sequence: each draft hangs on an earlier one, mostly a near one."""
    words = -(-max(new) // 32)
    mask = np.zeros((sum(new), words * 32), np.uint8)
    at = 0
    for n in new:
        for i in range(n):
            if i:
                mask[at + i] = mask[at + max(0, i - 1 - int(rng.exponential(4.0)))]
            mask[at + i, i] = 1
        at += n
    return torch.from_numpy(np.packbits(mask, axis=1, bitorder="little").view(np.int32).copy()).cuda()


def _prepare_tree(case, g):
    s, dt = _prepare_pages(case, g), DTYPES[case["dtype"]]
    h, hd = case["heads"], case["head_dim"]
    rng = np.random.default_rng(int(torch.randint(0, 1 << 30, (1,), generator=g, device="cuda")))
    s["mask"] = _draft_trees(_lengths(case)[0], rng)
    if case["gate"]:  # as the query projection gives them: each head's query, then its gate
        both = _normal(g, (s["rows"], h, 2, hd), dt, 1.5)
        s["q"], s["gate"] = both[:, :, 0], both[:, :, 1]
    else:
        s["q"] = _normal(g, (s["rows"], h, hd), dt, 1.5)
    s["out"] = torch.zeros(s["rows"], h, hd, dtype=dt, device="cuda")
    return s


def _prepare_commit(case, g):
    s = _prepare_pages(case, g, case["layers"])
    rng = np.random.default_rng(int(torch.randint(0, 1 << 30, (1,), generator=g, device="cuda")))
    new, most = _lengths(case)[0], case["accepted"]
    path, length = np.full((case["seqs"], most), -1, np.int32), np.zeros(case["seqs"], np.int32)
    for i, n in enumerate(new):  # the root, then drafts of which each lies past the path's length, as in a wide tree
        m = int(min(rng.integers(1, most + 1), max(1, n // 2)))
        rest = np.sort(rng.choice(np.arange(m, n), m - 1, replace=False)) if m > 1 else []
        path[i, :m], length[i] = [0, *rest], m
    s["path"], s["path_len"] = torch.from_numpy(path).cuda(), torch.from_numpy(length).cuda()
    s["lens_out"] = torch.zeros_like(s["lens"])
    return s


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    make = {"norm": _prepare_norm, "append": _prepare_append, "tables": _prepare_tables, "tree": _prepare_tree,
            "commit": _prepare_commit}[case["kind"]]
    return make(case, g) | {"case": case}


# ------------------------------------------------------------------------------------------------- plain forms
def _normed_rotated(x, weight, pos, dim, layout):
    """x [rows, heads, head_dim]: each head over its root mean square, times the weight, rotated; in 32 bits."""
    x = x.float()
    x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * weight
    i = torch.arange(dim // 2, device=pos.device, dtype=torch.float64)
    angle = pos.double()[:, None, None] * THETA ** (-2.0 * i / dim)
    cos, sin = torch.cos(angle).float(), torch.sin(angle).float()
    if layout == "half":
        a, b = x[..., :dim // 2], x[..., dim // 2:dim]
        turned = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    else:
        a, b = x[..., 0:dim:2], x[..., 1:dim:2]
        turned = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    return torch.cat([turned, x[..., dim:]], -1)


def _plain_norm(s):
    c = s["case"]
    return {"q": _normed_rotated(s["q"], s["q_weight"], s["pos"], c["dim"], c["layout"]).to(s["q"].dtype),
            "k": _normed_rotated(s["k"], s["k_weight"], s["pos"], c["dim"], c["layout"]).to(s["k"].dtype)}


def _plain_append(s):
    c = s["case"]
    rows = torch.arange(s["rows"], device="cuda")
    seq = torch.searchsorted(s["starts"][1:].long(), rows, right=True)
    pos = s["lens"].long()[seq] - s["starts"].long()[seq + 1] + rows
    page, slot = s["table"][seq, pos // c["page"]].long(), pos % c["page"]
    s["k"][page, slot] = _normed_rotated(s["new_k"], s["k_weight"], pos, c["dim"], c["layout"]).to(s["k"].dtype)
    s["v"][page, slot] = s["new_v"].to(s["v"].dtype)
    q = _normed_rotated(s["q"], s["q_weight"], pos, c["dim"], c["layout"]).to(s["q"].dtype)
    return {"q": q, "k": s["k"], "v": s["v"]}


def _plain_tables(s):
    c = s["case"]
    page, cols, n_pages = c["page"], s["pages"].shape[1], s["ring"].shape[0]
    first, free = s["state"][0].long(), s["state"][1].long()
    before, held, new = s["before"].long(), s["held"].long(), s["new"].long()
    rows, ended = new.clamp(min=0), new < 0
    lens = torch.where(ended, 0, before + rows)
    need = (lens + page - 1) // page
    want = need.clamp(max=cols)
    take, back = (want - held).clamp(min=0), (held - want).clamp(min=0)
    take_end, back_end = take.cumsum(0), back.cumsum(0)
    served = take_end <= free
    col = torch.arange(cols, device="cuda")
    grows = (col >= held[:, None]) & (col < want[:, None])
    from_ring = s["ring"][(first + (take_end - take)[:, None] + col - held[:, None]) % n_pages]
    pages = torch.where(grows, torch.where(served[:, None], from_ring, -1), s["pages"])
    goes = (col >= want[:, None]) & (col < held[:, None])
    to = (first + free + (back_end - back)[:, None] + col - want[:, None]) % n_pages
    s["ring"][to[goes]] = s["pages"][goes]
    s["pages"].copy_(pages)
    taken = torch.where(served, take, 0)
    starts = torch.cat([torch.zeros(1, dtype=torch.int64, device="cuda"), rows.cumsum(0)])
    r = torch.arange(s["rows"], device="cuda")
    seq = torch.searchsorted(starts[1:].contiguous(), r, right=True)
    pos = before[seq] + r - starts[seq]
    at = pages[seq, (pos // page).clamp(max=cols - 1)].long()
    slots = torch.where((pos // page < cols) & (at >= 0), at * page + pos % page, -1)
    return {"pages": s["pages"], "ring": s["ring"], "held": torch.where(served, want, torch.minimum(held, want)).int(),
            "state": torch.stack([(first + taken.sum()) % n_pages, free - taken.sum() + back_end[-1]]).int(),
            "starts": starts.int(), "lens": lens.int(), "missing": (need - want + torch.where(served, 0, take)).int(),
            "pos": pos.int(), "slots": slots}


def _mask_bits(mask):
    """Mask words [rows, words] as truth values [rows, 32 words]."""
    return ((mask[:, :, None] >> torch.arange(32, device=mask.device, dtype=torch.int32)) & 1).flatten(1).bool()


def _plain_tree(s):
    c = s["case"]
    n, kv, hd, g, m = c["seqs"], c["kv"], c["head_dim"], c["heads"] // c["kv"], s["most_new"]
    pages = s["table"].long().clamp(min=0)
    keys, values = (t[pages].reshape(n, -1, kv, hd)[:, :s["longest"]].float().transpose(1, 2).contiguous()
                    for t in (s["k"], s["v"]))  # [sequences, kv, positions, head_dim]
    starts, lens = s["starts"].long(), s["lens"].long()
    i = torch.arange(m, device="cuda")
    have = starts[1:] - starts[:-1]
    rows = (starts[:-1, None] + i).clamp(max=s["rows"] - 1)  # [sequences, new]
    q = s["q"][rows].float().reshape(n, m, kv, g, hd).permute(0, 2, 3, 1, 4).reshape(n, kv, g * m, hd)
    scores = (q @ keys.transpose(2, 3).contiguous() * (1.0 / math.sqrt(hd))).view(n, kv, g, m, -1)
    bits = _mask_bits(s["mask"])[rows]  # [sequences, new, new padded]
    base = (lens - have)[:, None, None]
    j = torch.arange(s["longest"], device="cuda")
    rel = (j - base).expand(n, m, -1)
    own_tree = torch.gather(bits, 2, rel.clamp(0, bits.shape[2] - 1)) & (rel < have[:, None, None])
    past = rel < 0
    if c["window"]:
        past &= j >= base + bits.sum(-1, keepdim=True) - c["window"]
    seen = torch.where(rel >= 0, own_tree, past)
    scores = scores.masked_fill_(~seen[:, None, None], float("-inf"))
    top = scores.amax(-1, keepdim=True)
    p = torch.exp(scores.sub_(torch.where(torch.isinf(top), 0.0, top)))
    total = p.sum(-1, keepdim=True)
    o = (p.view(n, kv, g * m, -1) @ values).view(n, kv, g, m, hd) / torch.where(total == 0, 1.0, total)
    o = o.permute(0, 3, 1, 2, 4).reshape(n, m, c["heads"], hd)[i < have[:, None]]  # rows in order
    if c["gate"]:
        o = o / (1.0 + torch.exp(-s["gate"].float()))
    return o.to(s["q"].dtype)


def _plain_commit(s):
    c = s["case"]
    starts, lens = s["starts"].long(), s["lens"].long()
    base = (lens - starts[1:] + starts[:-1])[:, None]
    i = torch.arange(s["path"].shape[1], device="cuda")
    kept = i < s["path_len"][:, None]
    seq = torch.arange(c["seqs"], device="cuda")[:, None].expand_as(kept)[kept]
    to, src = (base + i)[kept], (base + s["path"])[kept]
    page = lambda p: s["table"][seq, p // c["page"]].long()  # noqa: E731
    for pool in (s["k"], s["v"]):
        pool[:, page(to), to % c["page"]] = pool[:, page(src), src % c["page"]]
    return {"k": s["k"], "v": s["v"], "lens": (base[:, 0] + s["path_len"]).int()}


# --------------------------------------------------------------------------------------- the framework's calls
_kept = {}


def _package():
    """The package, a context on the device, and the stream a program queues its operators on."""
    if not _kept:
        at = os.path.join(os.getcwd(), "qwen-3.8-in-rust_amd")
        if at not in sys.path:
            sys.path.insert(0, at)
        import aqueduct as aq
        stream = torch.cuda.Stream()
        _kept.update(aq=aq, ctx=aq.Context(0), stream=stream, handle=stream.cuda_stream, ropes={}, workspace=None)
    return _kept["aq"], _kept["ctx"], _kept["handle"]


def _rope_of(dim, layout):
    """The rotation's table, made once as a model's program makes it."""
    aq, ctx, _ = _package()
    if (dim, layout) not in _kept["ropes"]:
        _kept["ropes"][dim, layout] = aq.Rope(ctx, dim, THETA, layout=layout)
    return _kept["ropes"][dim, layout]


def _type(name):
    aq, _, _ = _package()
    return {"f32": aq.F32, "f16": aq.F16, "bf16": aq.BF16}[name]


def _heads(t, name):
    aq, _, _ = _package()
    return aq.heads(t.data_ptr(), _type(name), t.stride(0), t.stride(1))


def _cache(s, k, v):
    aq, _, _ = _package()
    c = s["case"]
    return aq.paged_kv(k.data_ptr(), v.data_ptr(), _type(c["cache"]), k.shape[0], c["page"], c["kv"], c["head_dim"],
                       k.stride(0), k.stride(1), k.stride(2))


def _batch(s):
    aq, _, _ = _package()
    return aq.paged_batch(s["case"]["seqs"], s["starts"].data_ptr(), s["lens"].data_ptr(), s["table"].data_ptr(),
                          s["table"].shape[1], s["rows"], s["most_new"], s["longest"])


def _own_norm(s):
    aq, ctx, handle = _package()
    c, t = s["case"], s["case"]["dtype"]
    if "call" not in s:
        s["call"] = (ctx, _heads(s["q"], t), _heads(s["q_out"], t), c["heads"], _heads(s["k"], t), _heads(s["k_out"], t),
                     c["kv"], c["head_dim"], c["rows"], s["q_weight"].data_ptr(), s["k_weight"].data_ptr(), EPS,
                     _rope_of(c["dim"], c["layout"]), s["pos"].data_ptr(), handle)
    aq.qk_norm_rope(*s["call"])
    return {"q": s["q_out"], "k": s["k_out"]}


def _own_append(s):
    aq, ctx, handle = _package()
    c, t = s["case"], s["case"]["dtype"]
    if "call" not in s:
        s["call"] = (ctx, _cache(s, s["k"], s["v"]), _batch(s), _heads(s["new_k"], t), _heads(s["new_v"], t),
                     _heads(s["q"], t), _heads(s["q_out"], t), c["heads"], s["q_weight"].data_ptr(),
                     s["k_weight"].data_ptr(), EPS, _rope_of(c["dim"], c["layout"]), None, handle)
    aq.paged_append_norm(*s["call"])
    return {"q": s["q_out"], "k": s["k"], "v": s["v"]}


def _own_tables(s):
    aq, ctx, handle = _package()
    c = s["case"]
    if "call" not in s:
        t = aq.page_tables(c["seqs"], s["pages"].shape[1], s["ring"].shape[0], c["page"], s["pages"].data_ptr(),
                           s["held"].data_ptr(), s["ring"].data_ptr(), s["state"].data_ptr(),
                           held_out=s["held_out"].data_ptr(), free_state_out=s["state_out"].data_ptr())
        s["call"] = (ctx, t, s["before"].data_ptr(), s["new"].data_ptr(), s["rows"], s["starts"].data_ptr(),
                     s["lens"].data_ptr(), s["missing"].data_ptr(), s["pos"].data_ptr(), s["slots"].data_ptr(), None,
                     handle)
    aq.paged_tables(*s["call"])
    return {"pages": s["pages"], "ring": s["ring"], "held": s["held_out"], "state": s["state_out"][:2],
            "starts": s["starts"], "lens": s["lens"], "missing": s["missing"], "pos": s["pos"], "slots": s["slots"]}


def _own_tree(s):
    aq, ctx, handle = _package()
    c = s["case"]
    if "call" not in s:
        cache, batch = _cache(s, s["k"], s["v"]), _batch(s)
        need = aq.paged_attention_workspace(ctx, cache, batch, c["heads"])
        if _kept["workspace"] is None or _kept["workspace"].numel() < need:
            torch.cuda.synchronize()  # nothing queued still uses the smaller one
            _kept["workspace"] = torch.empty(need, dtype=torch.uint8, device="cuda")
        gate = _heads(s["gate"], c["dtype"]) if c["gate"] else None
        s["call"] = (ctx, cache, batch, s["mask"].data_ptr(), s["mask"].shape[1], c["heads"], _heads(s["q"], c["dtype"]),
                     _heads(s["out"], c["dtype"]), 1.0 / math.sqrt(c["head_dim"]), c["window"], gate)
    aq.paged_tree_attention(*s["call"], _kept["workspace"].data_ptr(), _kept["workspace"].numel(), handle)
    return s["out"]


def _own_commit(s):
    aq, ctx, handle = _package()
    if "call" not in s:
        caches = aq.paged_kv_array([_cache(s, k, v) for k, v in zip(s["k"], s["v"])])
        s["call"] = (ctx, caches, _batch(s), s["path"].data_ptr(), s["path_len"].data_ptr(), s["path"].shape[1],
                     s["lens_out"].data_ptr(), handle)
    aq.paged_tree_commit(*s["call"])
    return {"k": s["k"], "v": s["v"], "lens": s["lens_out"]}


def run(state):
    kind = state["case"]["kind"]
    if own:
        return {"norm": _own_norm, "append": _own_append, "tables": _own_tables, "tree": _own_tree,
                "commit": _own_commit}[kind](state)
    return {"norm": _plain_norm, "append": _plain_append, "tables": _plain_tables, "tree": _plain_tree,
            "commit": _plain_commit}[kind](state)


# -------------------------------------------------------------------------------------------------------- work
def work(case):
    kind = case["kind"]
    if kind == "tables":
        before, new, held, want, free, n_pages = _requests(case)
        moved = sum(abs(w - h) for w, h in zip(want, held))  # entries written, and read from the ring or the table
        rows = sum(max(n, 0) for n in new)
        return {"bytes": 4.0 * (8 * case["seqs"] + 2 * moved) + rows * (4 + 8), "flops": 0.0}
    hd, kv = case["head_dim"], case["kv"]
    if kind == "norm":
        values = case["rows"] * (case["heads"] + kv)
        return {"bytes": 2.0 * values * hd * ROW_BYTES[case["dtype"]] + 4 * case["rows"] + 8 * hd,
                "flops": values * (4.0 * hd + 3.0 * case["dim"])}
    new, lens = _lengths(case)
    rows, cache_b = sum(new), ROW_BYTES[case["cache"]]
    if kind == "commit":
        moved = sum(min(case["accepted"], max(1, n // 2)) for n in new) / 2.0  # about: paths differ by the seed
        return {"bytes": 4.0 * moved * case["layers"] * kv * hd * cache_b, "flops": 0.0}
    h, row_b = case["heads"], ROW_BYTES[case["dtype"]]
    if kind == "append":
        return {"bytes": float(rows * hd * (2 * h * row_b + 2 * kv * (row_b + cache_b))),
                "flops": rows * (h + kv) * (4.0 * hd + 3.0 * case["dim"])}
    window = case["window"] or max(lens)
    seen = sum(min(t - n, window) + n for n, t in zip(new, lens))
    pairs = sum(n * (min(t - n, window) + math.log2(n + 1)) for n, t in zip(new, lens))  # a few ancestors each
    return {"bytes": float(2 * seen * kv * hd * cache_b + (3 if case["gate"] else 2) * rows * h * hd * row_b),
            "flops": 4.0 * pairs * h * hd}


# ------------------------------------------------------------------------------------------------------- exact
def _turned(x, weight, pos, case):
    """Normed and rotated pair by pair as complex numbers, in 64 bits."""
    dim, half = case["dim"], case["dim"] // 2
    x = x.double()
    y = x / torch.sqrt((x ** 2).sum(-1, keepdim=True) / case["head_dim"] + EPS) * weight.double()
    freq = torch.tensor([math.exp(-2.0 * i / dim * math.log(THETA)) for i in range(half)], dtype=torch.float64,
                        device=x.device)
    angle = pos.double()[:, None, None] * freq
    first, second = (slice(0, half), slice(half, dim)) if case["layout"] == "half" else (slice(0, dim, 2),
                                                                                       slice(1, dim, 2))
    z = torch.complex(y[..., first], y[..., second]) * torch.polar(torch.ones_like(angle), angle)
    y[..., first], y[..., second] = z.real, z.imag
    return y


def exact(case, seed):
    if case["kind"] == "tables":
        return None  # whole numbers
    s = prepare(case, seed)
    if case["kind"] == "norm":
        return {"q": _turned(s["q"], s["q_weight"], s["pos"], case), "k": _turned(s["k"], s["k_weight"], s["pos"], case)}
    new, lens = _lengths(case)
    table, page, at = s["table"].cpu(), case["page"], 0
    if case["kind"] == "append":
        k, v, q = s["k"].double(), s["v"].double(), []
        for i, (n, total) in enumerate(zip(new, lens)):
            pos = torch.arange(total - n, total, device="cuda")
            places = torch.tensor([int(table[i, p // page]) * page + p % page for p in range(total - n, total)],
                                  device="cuda")
            k.view(-1, *k.shape[2:])[places] = _turned(s["new_k"][at:at + n], s["k_weight"], pos, case)
            v.view(-1, *v.shape[2:])[places] = s["new_v"][at:at + n].double()
            q.append(_turned(s["q"][at:at + n], s["q_weight"], pos, case))
            at += n
        return {"q": torch.cat(q), "k": k, "v": v}
    if case["kind"] == "commit":
        path, length = s["path"].cpu(), s["path_len"].cpu()
        for pool in (s["k"], s["v"]):
            for i, (n, total) in enumerate(zip(new, lens)):
                for e in range(int(length[i])):
                    a, b = total - n + e, total - n + int(path[i, e])
                    pool[:, table[i, a // page], a % page] = pool[:, table[i, b // page], b % page].clone()
        return {"k": s["k"].double(), "v": s["v"].double(), "lens": None}
    group, hd, out, mask = case["heads"] // case["kv"], case["head_dim"], [], _mask_bits(s["mask"])
    for i, (n, total) in enumerate(zip(new, lens)):
        used = table[i, :-(-total // page)].long().cuda()
        k, v = (t[used].flatten(0, 1)[:total].double() for t in (s["k"], s["v"]))
        hidden = torch.zeros(n, total, dtype=torch.bool, device="cuda")
        hidden[:, total - n:] = ~mask[at:at + n, :n]
        if case["window"]:
            j = torch.arange(total, device="cuda")
            first = total - n + mask[at:at + n].sum(-1, keepdim=True) - case["window"]
            hidden |= (j < first) & (j < total - n)
        o = torch.empty(n, case["heads"], hd, dtype=torch.float64, device="cuda")
        for h in range(case["heads"]):
            x = s["q"][at:at + n, h].double() @ k[:, h // group].T.contiguous() / math.sqrt(hd)
            o[:, h] = torch.softmax(x.masked_fill(hidden, -math.inf), -1) @ v[:, h // group].contiguous()
        if case["gate"]:
            o *= torch.sigmoid(s["gate"][at:at + n].double())
        out.append(o)
        at += n
    return torch.cat(out)
