"""Attention over a paged K/V cache and what feeds it, as cases that can be timed: rotary positions, new keys and values
appended to pages, and the new tokens of many sequences attending over their pages.

A case is a dict of plain values; its "kind" says which operator it runs:

  rope    rotate rows of heads by their positions, or back ("inverse": the rotation's gradient, and moving cached keys)
  append  write the new rows of a batch of sequences into their pages, keys rotated on the way and queries beside them
  attend  the new tokens of a batch of sequences over their pages: single tokens, verify batches, prompt chunks

`own` false: elementary torch operations in 32 bits (angles in 64), rounded once at the end. `own` true: the calls of the
`aqueduct` package, queued on the one stream that a program keeps.
"""
import math
import os
import sys

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
ROW_BYTES = {"f32": 4, "f16": 2, "bf16": 2}
THETA = 1e7
GOLDEN = 0.6180339887498949


# ------------------------------------------------------------------------------------------------------- cases
def rope(rows, heads, head_dim, dim, layout, scaling, dtype, inverse=False, first=0):
    return {"kind": "rope", "rows": rows, "heads": heads, "head_dim": head_dim, "dim": dim, "layout": layout,
            "scaling": scaling, "dtype": dtype, "inverse": inverse, "first": first}


def append(seqs, new, context, heads, kv, head_dim, dim, layout, page, dtype, cache):
    return {"kind": "append", "seqs": seqs, "new": new, "context": context, "heads": heads, "kv": kv,
            "head_dim": head_dim, "dim": dim, "layout": layout, "page": page, "dtype": dtype, "cache": cache}


def attend(seqs, new, context, heads, kv, head_dim, page, dtype, cache, window=0, gate=False):
    return {"kind": "attend", "seqs": seqs, "new": new, "context": context, "heads": heads, "kv": kv,
            "head_dim": head_dim, "page": page, "dtype": dtype, "cache": cache, "window": window, "gate": gate}


def listed():
    return [
        # the query and key heads of one token of the 27B shapes, a quarter of each head rotated: launch and latency
        dict(rope(1, 28, 256, 64, "half", "none", "f32", first=4097), name="rope_f32_1x28x256"),
        # a whole prompt of heads rotated in full, past the trained length
        dict(rope(8191, 40, 128, 128, "interleaved", "yarn", "bf16", first=60001), name="rope_bf16_8191x40x128_yarn"),
        # keys moved back, as when the front of a context is dropped; also the gradient of the rotation
        dict(rope(2001, 8, 128, 96, "half", "linear", "f16", inverse=True, first=70000),
             name="rope_f16_2001x8x128_back"),
        # one decode step of a served batch: a token for each of 48 sequences
        dict(append(48, 1, 4000, 32, 8, 128, 128, "half", 16, "bf16", "bf16"), name="append_bf16_48x1"),
        # ragged prompt chunks of four requests, f32 activations into a 16-bit cache
        dict(append(4, 1500, 900, 24, 4, 256, 64, "interleaved", 64, "f32", "f16"), name="append_f32_f16_4x1500"),
        # the first steps of a small model's decode: launch and latency
        dict(attend(1, 1, 50, 4, 2, 64, 16, "f32", "f32"), name="decode_f32_1_at_50"),
        # plain decode of one conversation in the 27B's heads
        dict(attend(1, 1, 8000, 24, 4, 256, 64, "f16", "f16"), name="decode_f16_1_at_8000"),
        # a decode step of a served batch, lengths far apart, small pages
        dict(attend(48, 1, 6000, 32, 8, 128, 16, "bf16", "bf16"), name="decode_bf16_48_at_6000"),
        # --spec 3 verify batches of eight conversations: f32 rows, half as much cache, the model's output gate
        dict(attend(8, 4, 3000, 24, 4, 256, 32, "f32", "f16", gate=True), name="verify_f32_f16_8x4_at_3000"),
        # a 64-row prompt chunk on the f32 cache
        dict(attend(1, 64, 4001, 24, 4, 256, 16, "f32", "f32"), name="chunk_f32_64_at_4001"),
        # a longer chunk of a document's prompt
        dict(attend(1, 512, 32000, 24, 4, 256, 64, "bf16", "bf16"), name="chunk_bf16_512_at_32000"),
        # whole prompts of three requests of different length
        dict(attend(3, 3500, 0, 32, 8, 128, 64, "f16", "f16"), name="prompt_f16_3x3500"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _draw_heads(rng):
    return rng.choice([(24, 4, 256), (24, 4, 256), (32, 8, 128), (28, 4, 128), (4, 2, 64), (16, 16, 64), (14, 2, 64),
                       (8, 1, 128), (16, 16, 80), (20, 4, 96), (16, 4, 192)])


def _draw_types(rng):
    return rng.choice([("f16", "f16"), ("bf16", "bf16"), ("f32", "f32"), ("f32", "f16"), ("f32", "bf16")])


def draw(rng):
    kind = rng.choice(["rope", "append", "attend", "attend", "attend"])
    page = rng.choice([16, 16, 32, 64, 128, 24])
    layout = rng.choice(["half", "interleaved"])
    heads, kv, hd = _draw_heads(rng)
    if kind == "rope":
        return rope(_log_int(rng, 1, 8000), rng.choice([kv, heads, heads + kv]), hd, rng.choice([hd, hd // 2, 32]),
                    layout, rng.choice(["none", "linear", "yarn"]), rng.choice(["f32", "f16", "bf16"]),
                    rng.random() < 0.3, _log_int(rng, 1, 200000))
    dtype, cache = _draw_types(rng)
    if kind == "append":
        seqs = _log_int(rng, 1, 64)
        return append(seqs, _log_int(rng, 1, max(2, 6000 // seqs)), _log_int(rng, 1, 4000), heads, kv, hd,
                      rng.choice([hd, hd // 2, 32]), layout, page, dtype, cache)
    if rng.random() < 0.6:
        seqs, new = _log_int(rng, 1, 48), rng.choice([1, 1, 1, 2, 4, 8])
        context = _log_int(rng, 10, min(16000, 170_000_000 // (seqs * kv * hd)))
    else:
        seqs, new = rng.randint(1, 4), _log_int(rng, 9, 1500 if dtype == "f32" else 3000)
        context = _log_int(rng, 1, min(16000, 250_000_000 // (seqs * new * heads)))
    return attend(seqs, new, context, heads, kv, hd, page, dtype, cache, rng.choice([0, 0, 0, _log_int(rng, 32, 4096)]),
                  rng.random() < 0.3)


def _ragged(mean, n, shift):
    """n whole numbers spread between a quarter and seven quarters of `mean`; one alone, or a mean of 1, is `mean`."""
    if n == 1 or mean <= 1:
        return [mean] * n
    return [max(1, int(mean * (0.25 + 1.5 * ((i * GOLDEN + shift) % 1.0)))) for i in range(n)]


def _lengths(case):
    """Each sequence's new rows, and its length with them."""
    new = _ragged(case["new"], case["seqs"], 0.5) if case["new"] > 8 else [case["new"]] * case["seqs"]
    before = _ragged(case["context"], case["seqs"], 0.25)
    return new, [a + b for a, b in zip(new, before)]


# ------------------------------------------------------------------------------------------------------ prepare
def _normal(g, shape, dtype, sigma=1.0):
    return (torch.randn(shape, generator=g, device="cuda") * sigma).to(dtype)


def _prepare_rope(case, g):
    dt = DTYPES[case["dtype"]]
    x = _normal(g, (case["rows"], case["heads"], case["head_dim"]), dt)
    jump = int(torch.randint(0, 4096, (1,), generator=g, device="cuda"))
    pos = torch.arange(case["rows"], device="cuda", dtype=torch.int32) + (case["first"] + jump)
    return {"x": x, "pos": pos, "y": torch.zeros_like(x)}


def _prepare_pages(case, g):
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
    return {"k": _normal(g, shape, ct), "v": _normal(g, shape, ct), "table": table.cuda(),
            "starts": torch.tensor(starts, dtype=torch.int32, device="cuda"),
            "lens": torch.tensor(lens, dtype=torch.int32, device="cuda"),
            "rows": starts[-1], "most_new": max(new), "longest": max(lens)}


def _prepare_append(case, g):
    s, dt = _prepare_pages(case, g), DTYPES[case["dtype"]]
    s["q"] = _normal(g, (s["rows"], case["heads"], case["head_dim"]), dt, 1.5)
    s["new_k"] = _normal(g, (s["rows"], case["kv"], case["head_dim"]), dt)
    s["new_v"] = _normal(g, (s["rows"], case["kv"], case["head_dim"]), dt)
    s["q_out"] = torch.zeros_like(s["q"])
    return s


def _prepare_attend(case, g):
    s, dt = _prepare_pages(case, g), DTYPES[case["dtype"]]
    h, hd = case["heads"], case["head_dim"]
    if case["gate"]:  # as the query projection gives them: each head's query, then its gate
        both = _normal(g, (s["rows"], h, 2, hd), dt, 1.5)
        s["q"], s["gate"] = both[:, :, 0], both[:, :, 1]
    else:
        s["q"] = _normal(g, (s["rows"], h, hd), dt, 1.5)
    s["out"] = torch.zeros(s["rows"], h, hd, dtype=dt, device="cuda")
    return s


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    make = {"rope": _prepare_rope, "append": _prepare_append, "attend": _prepare_attend}[case["kind"]]
    return make(case, g) | {"case": case}


# ------------------------------------------------------------------------------------------------- plain forms
SCALED = {"none": {}, "linear": {"factor": 4.0}, "yarn": {"factor": 8.0, "orig_ctx": 32768}}
BETA_FAST, BETA_SLOW = 32.0, 1.0


def _angles(pos, dim, scaling):
    """(cos, sin) [rows, dim / 2] of the positions, angles in 64 bits."""
    i = torch.arange(dim // 2, device=pos.device, dtype=torch.float64)
    freq = THETA ** (-2.0 * i / dim)
    gain = 1.0
    if scaling == "linear":
        freq = freq / SCALED["linear"]["factor"]
    elif scaling == "yarn":
        factor, orig = SCALED["yarn"]["factor"], SCALED["yarn"]["orig_ctx"]
        lo, hi = (dim * math.log(orig / (2 * math.pi * b)) / (2 * math.log(THETA)) for b in (BETA_FAST, BETA_SLOW))
        lo, hi = max(math.floor(lo), 0), min(math.ceil(hi), dim - 1)
        kept = 1.0 - ((i - lo) / max(hi - lo, 1e-3)).clamp(0, 1)
        freq = freq / factor * (1 - kept) + freq * kept
        gain = 0.1 * math.log(factor) + 1.0
    a = pos.double()[:, None] * freq
    return torch.cos(a) * gain, torch.sin(a) * gain


def _rotated(x, pos, dim, layout, scaling, inverse=False):
    """x [rows, heads, head_dim] rotated, in 32 bits."""
    cos, sin = (t.float()[:, None, :] for t in _angles(pos, dim, scaling))
    if inverse:
        sin = -sin
    x = x.float()
    if layout == "half":
        a, b = x[..., :dim // 2], x[..., dim // 2:dim]
        turned = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    else:
        a, b = x[..., 0:dim:2], x[..., 1:dim:2]
        turned = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    return torch.cat([turned, x[..., dim:]], -1)


def _plain_rope(s):
    c = s["case"]
    return _rotated(s["x"], s["pos"], c["dim"], c["layout"], c["scaling"], c["inverse"]).to(s["x"].dtype)


def _places(s):
    """Sequence and position of each new row."""
    rows = torch.arange(s["rows"], device="cuda")
    seq = torch.searchsorted(s["starts"][1:].long(), rows, right=True)
    return seq, s["lens"].long()[seq] - s["starts"].long()[seq + 1] + rows


def _plain_append(s):
    c = s["case"]
    seq, pos = _places(s)
    page, slot = s["table"][seq, pos // c["page"]].long(), pos % c["page"]
    s["k"][page, slot] = _rotated(s["new_k"], pos, c["dim"], c["layout"], "none").to(s["k"].dtype)
    s["v"][page, slot] = s["new_v"].to(s["v"].dtype)
    q = _rotated(s["q"], pos, c["dim"], c["layout"], "none").to(s["q"].dtype)
    return {"q": q, "k": s["k"], "v": s["v"]}


def _plain_attend(s):
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
    at = (lens - have)[:, None] + i  # position of each new row
    j = torch.arange(s["longest"], device="cuda")
    seen = j <= at[..., None]
    if c["window"]:
        seen &= j > at[..., None] - c["window"]
    scores = scores.masked_fill_(~seen[:, None, None], float("-inf"))
    p = torch.exp(scores.sub_(scores.amax(-1, keepdim=True)))
    total = p.sum(-1, keepdim=True)
    o = (p.view(n, kv, g * m, -1) @ values).view(n, kv, g, m, hd) / total
    o = o.permute(0, 3, 1, 2, 4).reshape(n, m, c["heads"], hd)[i < have[:, None]]  # rows in order
    if c["gate"]:
        o = o / (1.0 + torch.exp(-s["gate"].float()))
    return o.to(s["q"].dtype)


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


def _rope_of(dim, layout, scaling):
    """The rotation's table, made once as a model's program makes it."""
    aq, ctx, _ = _package()
    key = (dim, layout, scaling)
    if key not in _kept["ropes"]:
        _kept["ropes"][key] = aq.Rope(ctx, dim, THETA, layout=layout, scaling=scaling, **SCALED[scaling])
    return _kept["ropes"][key]


def _heads(t, name):
    aq, _, _ = _package()
    return aq.heads(t.data_ptr(), {"f32": aq.F32, "f16": aq.F16, "bf16": aq.BF16}[name], t.stride(0), t.stride(1))


def _paged(s):
    aq, _, _ = _package()
    c, k = s["case"], s["k"]
    cache = aq.paged_kv(k.data_ptr(), s["v"].data_ptr(), {"f32": aq.F32, "f16": aq.F16, "bf16": aq.BF16}[c["cache"]],
                        k.shape[0], c["page"], c["kv"], c["head_dim"], k.stride(0), k.stride(1), k.stride(2))
    batch = aq.paged_batch(c["seqs"], s["starts"].data_ptr(), s["lens"].data_ptr(), s["table"].data_ptr(),
                           s["table"].shape[1], s["rows"], s["most_new"], s["longest"])
    return cache, batch


def _own_rope(s):
    aq, _, handle = _package()
    c = s["case"]
    if "call" not in s:
        s["call"] = (_rope_of(c["dim"], c["layout"], c["scaling"]), _heads(s["x"], c["dtype"]),
                     _heads(s["y"], c["dtype"]), c["rows"], c["heads"], c["head_dim"], s["pos"].data_ptr(),
                     c["inverse"], handle)
    aq.rope_apply(*s["call"])
    return s["y"]


def _own_append(s):
    aq, ctx, handle = _package()
    c = s["case"]
    if "call" not in s:
        s["call"] = (ctx, *_paged(s), _heads(s["new_k"], c["dtype"]), _heads(s["new_v"], c["dtype"]),
                     _rope_of(c["dim"], c["layout"], "none"), _heads(s["q"], c["dtype"]),
                     _heads(s["q_out"], c["dtype"]), c["heads"], handle)
    aq.paged_append(*s["call"])
    return {"q": s["q_out"], "k": s["k"], "v": s["v"]}


def _own_attend(s):
    aq, ctx, handle = _package()
    c = s["case"]
    if "call" not in s:
        cache, batch = _paged(s)
        need = aq.paged_attention_workspace(ctx, cache, batch, c["heads"])
        if _kept["workspace"] is None or _kept["workspace"].numel() < need:
            torch.cuda.synchronize()  # nothing queued still uses the smaller one
            _kept["workspace"] = torch.empty(need, dtype=torch.uint8, device="cuda")
        gate = _heads(s["gate"], c["dtype"]) if c["gate"] else None
        s["call"] = (ctx, cache, batch, c["heads"], _heads(s["q"], c["dtype"]), _heads(s["out"], c["dtype"]),
                     1.0 / math.sqrt(c["head_dim"]), c["window"], gate)
    aq.paged_attention(*s["call"], _kept["workspace"].data_ptr(), _kept["workspace"].numel(), handle)
    return s["out"]


def run(state):
    kind = state["case"]["kind"]
    if own:
        return {"rope": _own_rope, "append": _own_append, "attend": _own_attend}[kind](state)
    return {"rope": _plain_rope, "append": _plain_append, "attend": _plain_attend}[kind](state)


# -------------------------------------------------------------------------------------------------------- work
def work(case):
    hd, kind = case["head_dim"], case["kind"]
    if kind == "rope":
        values = case["rows"] * case["heads"]
        return {"bytes": 2.0 * values * hd * ROW_BYTES[case["dtype"]] + 4 * case["rows"],
                "flops": 3.0 * values * case["dim"]}
    new, lens = _lengths(case)
    rows, h, kv = sum(new), case["heads"], case["kv"]
    row_b, cache_b = ROW_BYTES[case["dtype"]], ROW_BYTES[case["cache"]]
    if kind == "append":
        return {"bytes": float(rows * hd * (2 * h * row_b + 2 * kv * (row_b + cache_b))),
                "flops": 3.0 * rows * (h + kv) * case["dim"]}
    window = case["window"] or max(lens)
    seen = pairs = 0
    for n, total in zip(new, lens):
        first = total - n  # position of the first new row
        seen += total - max(0, first + 1 - window)
        full = max(0, min(n, window - first))  # rows that see everything before them
        pairs += full * first + full * (full + 1) // 2 + (n - full) * window
    return {"bytes": float(2 * seen * kv * hd * cache_b + (3 if case["gate"] else 2) * rows * h * hd * row_b),
            "flops": 4.0 * pairs * h * hd}


# ------------------------------------------------------------------------------------------------------- exact
def _turn(x, pos, case, scaling, inverse=False):
    """The rotation by its matrix, pair by pair as complex numbers in 64 bits."""
    dim, half = case["dim"], case["dim"] // 2
    freq = torch.tensor([_frequency(i, dim, scaling) for i in range(half)], dtype=torch.float64, device=x.device)
    angle = pos.double()[:, None, None] * freq
    gain = 1.0 + 0.1 * math.log(SCALED["yarn"]["factor"]) if scaling == "yarn" else 1.0
    unit = torch.polar(torch.full_like(angle, gain), -angle if inverse else angle)
    y = x.double().clone()
    first, second = (slice(0, half), slice(half, dim)) if case["layout"] == "half" else (slice(0, dim, 2),
                                                                                       slice(1, dim, 2))
    z = torch.complex(y[..., first], y[..., second]) * unit
    y[..., first], y[..., second] = z.real, z.imag
    return y


def _frequency(i, dim, scaling):
    f = math.exp(-2.0 * i / dim * math.log(THETA))
    if scaling == "linear":
        return f / SCALED["linear"]["factor"]
    if scaling == "yarn":
        def index(turns):  # the pair that makes so many turns over the trained length
            return dim / 2 * math.log(SCALED["yarn"]["orig_ctx"] / (turns * 2 * math.pi)) / math.log(THETA)
        lo, hi = max(0, math.floor(index(BETA_FAST))), min(dim - 1, math.ceil(index(BETA_SLOW)))
        scaled = 0.0 if i <= lo else 1.0 if i >= hi else (i - lo) / (hi - lo)
        return f * (1 - scaled) + f / SCALED["yarn"]["factor"] * scaled
    return f


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "rope":
        return _turn(s["x"], s["pos"], case, case["scaling"], case["inverse"])
    new, lens = _lengths(case)
    table, page = s["table"].cpu(), case["page"]
    if case["kind"] == "append":
        k, v, q, at = s["k"].double(), s["v"].double(), [], 0
        for i, (n, total) in enumerate(zip(new, lens)):
            pos = torch.arange(total - n, total, device="cuda")
            places = torch.tensor([int(table[i, p // page]) * page + p % page for p in range(total - n, total)],
                                  device="cuda")
            k.view(-1, *k.shape[2:])[places] = _turn(s["new_k"][at:at + n], pos, case, "none")
            v.view(-1, *v.shape[2:])[places] = s["new_v"][at:at + n].double()
            q.append(_turn(s["q"][at:at + n], pos, case, "none"))
            at += n
        return {"q": torch.cat(q), "k": k, "v": v}
    group, hd, out, at = case["heads"] // case["kv"], case["head_dim"], [], 0
    for i, (n, total) in enumerate(zip(new, lens)):
        used = table[i, :-(-total // page)].long().cuda()
        k, v = (t[used].flatten(0, 1)[:total].double() for t in (s["k"], s["v"]))
        pos = torch.arange(total - n, total, device="cuda")[:, None]
        j = torch.arange(total, device="cuda")
        hidden = (j > pos) | (j <= pos - (case["window"] or total))
        o = torch.empty(n, case["heads"], hd, dtype=torch.float64, device="cuda")
        for h in range(case["heads"]):
            x = s["q"][at:at + n, h].double() @ k[:, h // group].T.contiguous() / math.sqrt(hd)
            o[:, h] = torch.softmax(x.masked_fill(hidden, -math.inf), -1) @ v[:, h // group].contiguous()
        if case["gate"]:
            o *= torch.sigmoid(s["gate"][at:at + n].double())
        out.append(o)
        at += n
    return torch.cat(out)
