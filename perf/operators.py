"""Operators of a server's step over paged caches, in their plain form and through the framework's kernels.

``rotary``: heads turned by their rows' positions.  ``append``: new keys and values of several sequences go to their pages, keys
and queries turned on the way.  ``attention``: the queries of those rows over the pages, one token or a chunk of each sequence.

A step's rows are those of its sequences one after the other: rows starts[s] .. starts[s + 1] - 1 are of sequence s and stand at
its last positions, the last one at lengths[s] - 1.  table[s][b] is the page that holds positions b * page ... of sequence s; pages
are [page index][kv head][slot][head dimension, padded]."""
import math
import os
import random
import sys

import torch

if os.getcwd() not in sys.path:
    sys.path.insert(0, os.getcwd())

own = False
DEVICE = "cuda"
F32, F64 = torch.float32, torch.float64
TYPE = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
_context = []


def framework():
    """The package, the program's one device context and its kernels."""
    if not _context:
        from __graft_entry__ import load_package
        pkg = load_package()
        ctx = pkg.Context(0)
        _context.extend((pkg, ctx, pkg.Kernels(ctx)))
    return _context


# ---- the cases ----------------------------------------------------------------------------------------------------------
def listed():
    gqa = {"heads": 32, "kv_heads": 8, "dim": 128, "page": 16, "dtype": "bf16"}
    rot = {"rot": 128, "first": 0, "halves": True, "base": 1e6, "stretch": 1.0, "amplitude": 1.0}
    return [
        # rotary positions -------------------------------------------------------------------------------------------------
        # one token's query heads: a launch's own time
        {"name": "rotary token", "op": "rotary", "rows": 1, "heads": 32, "dim": 128, "dtype": "bf16", "far": 32768, "margin": 2048, "layout": 1, **rot},
        # a long prompt's query heads, as the stacked projection leaves them
        {"name": "rotary prompt", "op": "rotary", "rows": 16384, "heads": 32, "dim": 128, "dtype": "bf16", "far": 16384, "margin": 2048, "layout": 2, **rot},
        # a run in 32 bits: neighbouring pairs in the last part of heads of an odd size, a context stretched four times
        {"name": "rotary part", "op": "rotary", "rows": 1001, "heads": 5, "dim": 80, "dtype": "f32", "far": 131072, "margin": 0, "layout": 3, "rot": 50, "first": 30,
         "halves": False, "base": 1e4, "stretch": 4.0, "amplitude": 1.1386},
        # appending to a paged cache ----------------------------------------------------------------------------------------
        # a server's step: one token of each of its sequences
        {"name": "append step of 64", "op": "append", "chunks": 0, "rows": 1, "tokens": 64, "context": 8000, "ragged": True, "layout": 4, **gqa, **rot},
        # a few prompts of different lengths in one pass, half precision, half of each head turned
        {"name": "append prompts", "op": "append", "chunks": 5, "rows": 1500, "tokens": 3, "context": 700, "ragged": True, "layout": 5, "heads": 16, "kv_heads": 4, "dim": 128,
         "page": 32, "dtype": "f16", "rot": 64, "first": 0, "halves": False, "base": 1e4, "stretch": 1.0, "amplitude": 1.0},
        # a whole long prompt
        {"name": "append long prompt", "op": "append", "chunks": 1, "rows": 16384, "tokens": 0, "context": 0, "ragged": False, "layout": 6, **gqa, **rot},
        # attention over a paged cache -----------------------------------------------------------------------------------------
        # one token of a chat with a long history: latency
        {"name": "attention token", "op": "attention", "chunks": 0, "rows": 1, "tokens": 1, "context": 32768, "ragged": False, "window": 0, "sink": False, "layout": 7, **gqa},
        # a server's step over sequences that are not equally long: memory
        {"name": "attention step of 64", "op": "attention", "chunks": 0, "rows": 1, "tokens": 64, "context": 16384, "ragged": True, "window": 0, "sink": False, "layout": 8,
         **gqa},
        # a portion of a long prompt at its end
        {"name": "attention chunk", "op": "attention", "chunks": 1, "rows": 512, "tokens": 0, "context": 16000, "ragged": False, "window": 0, "sink": False, "layout": 9, **gqa},
        # whole prompts of different lengths in one pass
        {"name": "attention prompts", "op": "attention", "chunks": 4, "rows": 4096, "tokens": 0, "context": 0, "ragged": True, "window": 0, "sink": False, "layout": 10,
         "heads": 16, "kv_heads": 4, "dim": 128, "page": 64, "dtype": "f16"},
        # a pass that brings prompts' portions beside other sequences' tokens, in a layer with a sliding window
        {"name": "attention window", "op": "attention", "chunks": 3, "rows": 256, "tokens": 29, "context": 8192, "ragged": True, "window": 512, "sink": False, "layout": 11,
         "heads": 8, "kv_heads": 1, "dim": 256, "page": 32, "dtype": "bf16"},
        # a reference run in 32 bits, with a learned sink
        {"name": "attention in 32 bits", "op": "attention", "chunks": 1, "rows": 333, "tokens": 2, "context": 100, "ragged": False, "window": 0, "sink": True, "layout": 12,
         "heads": 8, "kv_heads": 4, "dim": 64, "page": 16, "dtype": "f32"},
    ]


def spread(rng, lo, hi):
    """A whole number from lo to hi, evenly over the logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw_rotation(rng, dim):
    rot = rng.choice([dim, dim, dim // 2, 2 * rng.randint(1, dim // 2)])
    rot -= rot % 2
    stretch = rng.choice([1.0, 1.0, 4.0, 8.0])
    return {"rot": rot, "first": rng.choice([0, 0, dim - rot]), "halves": rng.random() < 0.6, "base": rng.choice([1e4, 1e6]), "stretch": stretch,
            "amplitude": 1.0 if stretch == 1.0 else 0.1 * math.log(stretch) + 1.0}


def draw(rng):
    op = rng.choice(["rotary", "append", "attention", "attention"])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    dim = rng.choice([64, 128, 128, 256, rng.randint(4, 32) * 8, rng.randint(32, 256) // 2 * 2])
    kv_heads = rng.choice([1, 2, 4, 8])
    heads = kv_heads * rng.choice([1, 2, 3, 4, 8])
    c = {"op": op, "heads": heads, "dim": dim, "dtype": dtype, "layout": rng.randrange(1 << 20)}
    if op == "rotary":
        values = 16384 * 32 * 128 // (2 if dtype == "f32" else 1)
        c.update(rows=spread(rng, 1, min(16384, values // (heads * dim))), far=spread(rng, 512, 1 << 20), margin=rng.choice([0, 0, dim, 1024]), **draw_rotation(rng, dim))
        return c
    c.update(kv_heads=kv_heads, page=rng.choice([16, 16, 32, 64, 128]))
    mode = rng.choice(["tokens", "chunks", "mixed"])
    c["tokens"] = 0 if mode == "chunks" else spread(rng, 1, 64)
    c["chunks"] = 0 if mode == "tokens" else rng.randint(1, 4)
    c["ragged"] = rng.random() < 0.7
    if op == "append":
        values = 16384 * 48 * 128 // (2 if dtype == "f32" else 1)
        most = min(16384, values // ((heads + 2 * kv_heads) * dim))
        c.update(rows=spread(rng, 1, max(1, most // max(c["chunks"], 1) - 64)) if c["chunks"] else 1, context=spread(rng, 1, 4000), **draw_rotation(rng, dim))
        return c
    c.update(window=rng.choice([0, 0, 0, spread(rng, 1, 2048)]), sink=rng.random() < 0.25)
    c.update(rows=spread(rng, 1, 2048) if c["chunks"] else 1, context=spread(rng, 1, 32768))
    while work(c)["bytes"] > (5e8 if dtype == "f32" else 2.5e9) or work(c)["flops"] > (4e9 if dtype == "f32" else 1.5e11):
        c["rows"], c["context"] = max(1, c["rows"] * 2 // 3), max(1, c["context"] * 2 // 3)
    return c


def sequences(c):
    """[(new rows, positions before them)] of the step's sequences: the chunks, then the single tokens."""
    r = random.Random(c["layout"])
    out = []
    for i in range(c["chunks"] + c["tokens"]):
        n = 1 if i >= c["chunks"] else r.randint((c["rows"] + 1) // 2, c["rows"]) if c["ragged"] else c["rows"]
        out.append((n, r.randint(c["context"] // 4, c["context"]) if c["ragged"] else c["context"]))
    return out


def padded(dim):
    """The columns of a head in the cache's pages."""
    return next(p for p in (32, 64, 128, 192, 256) if dim <= p)


# ---- seeded inputs ------------------------------------------------------------------------------------------------------
def normal(g, *shape, dtype=F32):
    return torch.randn(*shape, generator=g, device=DEVICE, dtype=dtype)


def frequencies(c):
    """f32, as a program keeps them: base^(-2i / rot), the slow half of them stretched for a longer context."""
    i = torch.arange(c["rot"] // 2, dtype=F64)
    f = c["base"] ** (-2.0 * i / c["rot"])
    ramp = (i / max(c["rot"] // 2 - 1, 1)).clamp(0, 1)
    return (f * (1 - ramp) + f / c["stretch"] * ramp).to(F32).to(DEVICE)


def words(values):
    return torch.tensor(values, dtype=torch.int32, device=DEVICE)


def rotary_inputs(c, seed):
    """Heads in the rows of a stacked projection, `margin` columns on each side of them, and the rows' positions."""
    g = torch.Generator(device=DEVICE).manual_seed(seed)
    r = random.Random(c["layout"])
    x = normal(g, c["rows"], c["heads"] * c["dim"] + 2 * c["margin"]).to(TYPE[c["dtype"]])
    at = []
    while len(at) < c["rows"]:                              # of a few sequences
        n = min(c["rows"] - len(at), max(1, c["rows"] // r.randint(1, 4)))
        first = r.randint(0, max(c["far"] - n, 0))
        at.extend(range(first, first + n))
    return {"x": x, "positions": words(at), "frequencies": frequencies(c)}


def step_inputs(c):
    """The step's sequences and their pages, which stand in the pool in no order."""
    seqs = sequences(c)
    need = [-(-(n + past) // c["page"]) for n, past in seqs]
    g = torch.Generator().manual_seed(c["layout"])
    pages = sum(need) + 3
    order, table, at = torch.randperm(pages, generator=g).tolist(), [], 0
    for n in need:
        table.append(order[at:at + n] + [0] * (max(need) - n))
        at += n
    starts = [0]
    for n, _ in seqs:
        starts.append(starts[-1] + n)
    return {"seqs": seqs, "pages": pages, "table": words(table), "starts": words(starts), "lengths": words([n + past for n, past in seqs]),
            "rows": starts[-1], "max_rows": max(n for n, _ in seqs), "max_length": max(n + past for n, past in seqs)}


def pool(c, s, g):
    """Pages with what earlier steps have left there; the columns behind a head's are zero."""
    p = torch.zeros(s["pages"], c["kv_heads"], c["page"], padded(c["dim"]), device=DEVICE, dtype=TYPE[c["dtype"]])
    for lo in range(0, s["pages"], 4096):
        part = p[lo:lo + 4096]
        part[..., :c["dim"]] = normal(g, *part.shape[:3], c["dim"]).to(p.dtype)
    return p


def append_inputs(c, seed):
    s, g = step_inputs(c), torch.Generator(device=DEVICE).manual_seed(seed)
    s["qkv"] = normal(g, s["rows"], (c["heads"] + 2 * c["kv_heads"]) * c["dim"]).to(TYPE[c["dtype"]])
    s["keys"], s["values"], s["frequencies"] = pool(c, s, g), pool(c, s, g), frequencies(c)
    return s


def attention_inputs(c, seed):
    s, g = step_inputs(c), torch.Generator(device=DEVICE).manual_seed(seed)
    s["q"] = normal(g, s["rows"], c["heads"], c["dim"]).to(TYPE[c["dtype"]])
    s["keys"], s["values"] = pool(c, s, g), pool(c, s, g)
    s["sink"] = normal(g, c["heads"]) if c["sink"] else None
    s["scale"] = c["dim"] ** -0.5
    return s


INPUTS = {"rotary": rotary_inputs, "append": append_inputs, "attention": attention_inputs}


def wrap(t, offset=0):
    """A buffer over a tensor's memory, `offset` values from its start."""
    pkg, ctx, _ = framework()
    size = t.element_size()
    return pkg.Buffer.wrap(ctx, t.data_ptr() + offset * size, (t.numel() - offset) * size, owner=t)


def prepare(case, seed):
    c = case
    s = INPUTS[c["op"]](c, seed)
    s["case"] = c
    if c["op"] == "rotary":
        s["out"] = torch.empty(c["rows"], c["heads"], c["dim"], device=DEVICE, dtype=s["x"].dtype)
    elif c["op"] == "append":
        s["out"] = torch.empty(s["rows"], c["heads"], c["dim"], device=DEVICE, dtype=s["qkv"].dtype)
    else:
        s["out"] = torch.empty_like(s["q"])
    if own:                                                 # what a program holds beside its data: buffers, an open batch, scratch memory
        pkg, ctx, K = framework()
        s["dtype"] = {"bf16": pkg.BF16, "f16": pkg.F16, "f32": pkg.F32}[c["dtype"]]
        s["batch"], b = pkg.CommandBatch(ctx), {}
        names = ["out", "positions", "frequencies", "keys", "values", "table", "starts", "lengths", "q", "sink"]
        for name in names:
            b[name] = wrap(s[name]) if s.get(name) is not None else None
        if c["op"] == "rotary":
            b["x"] = wrap(s["x"], c["margin"])
        elif c["op"] == "append":
            b["q"], b["k"], b["v"] = (wrap(s["qkv"], h * c["dim"]) for h in (0, c["heads"], c["heads"] + c["kv_heads"]))
        else:
            n = K.paged_attention_workspace_bytes(s["rows"], len(s["seqs"]), s["max_rows"], s["max_length"], c["heads"], c["kv_heads"], c["dim"])
            b["workspace"] = pkg.Buffer.empty(ctx, max(n, 16))
        s["buffers"] = b
    torch.cuda.synchronize()
    return s


# ---- through the framework ----------------------------------------------------------------------------------------------
def own_rotary(s):
    (pkg, _, K), c, b = framework(), s["case"], s["buffers"]
    K.rotary_rows_into(s["batch"], b["x"], b["out"], s["dtype"], b["positions"], b["frequencies"], c["amplitude"], c["rows"], c["heads"], c["dim"], c["rot"], c["first"],
                       pkg.ROTARY_HALVES if c["halves"] else pkg.ROTARY_PAIRS, s["x"].shape[1], c["heads"] * c["dim"])
    return s["out"]


def own_append(s):
    (pkg, _, K), c, b = framework(), s["case"], s["buffers"]
    ld = s["qkv"].shape[1]
    K.paged_append_into(s["batch"], b["k"], b["v"], s["dtype"], b["keys"], b["values"], b["table"], b["starts"], b["lengths"], s["rows"], len(s["seqs"]), c["kv_heads"],
                        c["dim"], s["pages"], c["page"], s["table"].shape[1], ld, ld, b["frequencies"], c["amplitude"], c["rot"], c["first"],
                        pkg.ROTARY_HALVES if c["halves"] else pkg.ROTARY_PAIRS, b["q"], b["out"], c["heads"], ld, c["heads"] * c["dim"])
    return [s["out"], s["keys"], s["values"]]


def own_attention(s):
    (_, _, K), c, b = framework(), s["case"], s["buffers"]
    ld = c["heads"] * c["dim"]
    K.paged_attention_into(s["batch"], b["q"], b["keys"], b["values"], b["out"], s["dtype"], b["table"], b["starts"], b["lengths"], s["rows"], len(s["seqs"]), s["max_rows"],
                           s["max_length"], c["heads"], c["kv_heads"], c["dim"], s["pages"], c["page"], s["table"].shape[1], ld, ld, s["scale"], c["window"], b["sink"],
                           b["workspace"])
    return s["out"]


# ---- plain forms --------------------------------------------------------------------------------------------------------
def turned(x, positions, s):
    """x [rows, heads, dim], its rotated columns turned; angles in 64 bits, the rest in 32."""
    c = s["case"]
    angle = positions.to(F64)[:, None] * s["frequencies"].to(F64)
    cos, sin = (angle.cos() * c["amplitude"]).to(F32)[:, None], (angle.sin() * c["amplitude"]).to(F32)[:, None]
    y = x.to(F32)
    first, rot = c["first"], c["rot"]
    part = y[..., first:first + rot]
    a, b = (part[..., :rot // 2], part[..., rot // 2:]) if c["halves"] else (part[..., 0::2], part[..., 1::2])
    u, v = a * cos - b * sin, b * cos + a * sin
    new = torch.cat([u, v], -1) if c["halves"] else torch.stack([u, v], -1).flatten(-2)
    return torch.cat([y[..., :first], new, y[..., first + rot:]], -1).to(x.dtype)


def plain_rotary(s):
    c = s["case"]
    n = c["heads"] * c["dim"]
    return turned(s["x"][:, c["margin"]:c["margin"] + n].unflatten(1, (c["heads"], c["dim"])), s["positions"], s)


def slots(s):
    """Position, page and slot of every row."""
    c = s["case"]
    starts, lengths = s["starts"].long(), s["lengths"].long()
    n = starts[1:] - starts[:-1]
    row = torch.arange(s["rows"], device=DEVICE)
    of = torch.searchsorted(starts, row, right=True) - 1
    position = lengths[of] - n[of] + row - starts[of]
    return position, s["table"].long()[of, position // c["page"]], position % c["page"]


def plain_append(s):
    c = s["case"]
    H, G, d = c["heads"], c["kv_heads"], c["dim"]
    position, page, slot = slots(s)
    heads = s["qkv"].unflatten(1, (H + 2 * G, d))
    q = turned(heads[:, :H], position, s)
    for target, x in ((s["keys"], turned(heads[:, H:H + G], position, s)), (s["values"], heads[:, H + G:])):
        target[page, :, slot] = torch.nn.functional.pad(x, (0, target.shape[3] - d))
    return [q, s["keys"], s["values"]]


def gathered(p, s, i, lo, hi, dim):
    """Positions lo .. hi - 1 of sequence i as [kv heads, positions, dim] in 32 bits."""
    size = p.shape[2]
    rows = p[s["table"][i, lo // size:-(-hi // size)].long()].transpose(0, 1).flatten(1, 2)
    return rows[:, lo % size:lo % size + hi - lo, :dim].to(F32)


def plain_attention(s):
    c = s["case"]
    H, G, d, row = c["heads"], c["kv_heads"], c["dim"], 0
    out = torch.empty_like(s["q"])
    for i, (n, past) in enumerate(s["seqs"]):
        hi = n + past
        lo = max(0, past + 1 - c["window"]) if c["window"] else 0
        k, v = (gathered(p, s, i, lo, hi, d) for p in (s["keys"], s["values"]))
        at, own_at = torch.arange(lo, hi, device=DEVICE), torch.arange(past, hi, device=DEVICE)[:, None]
        hidden = at > own_at
        if c["window"]:
            hidden |= at <= own_at - c["window"]
        q = s["q"][row:row + n].to(F32).unflatten(1, (G, H // G)).permute(1, 2, 0, 3)            # [kv head, head of it, row, dim]
        for g in range(G):
            z = (q[g] @ k[g].T * s["scale"]).masked_fill(hidden, -math.inf)
            top = z.amax(-1, keepdim=True)
            if s["sink"] is not None:
                own_sink = s["sink"][g * (H // G):(g + 1) * (H // G), None, None]
                top = torch.maximum(top, own_sink)
            w = (z - top).exp()
            total = w.sum(-1, keepdim=True)
            if s["sink"] is not None:
                total = total + (own_sink - top).exp()
            out[row:row + n, g * (H // G):(g + 1) * (H // G)] = ((w @ v[g]) / total).transpose(0, 1).to(out.dtype)
        row += n
    return out


RUN = {"rotary": (plain_rotary, own_rotary), "append": (plain_append, own_append), "attention": (plain_attention, own_attention)}


def run(state):
    return RUN[state["case"]["op"]][1 if own else 0](state)


# ---- what a pass cannot do without --------------------------------------------------------------------------------------
def visible(n, past, window):
    """(pairs of a row and a position that it sees, positions that some row sees)."""
    if not window:
        return n * past + n * (n + 1) // 2, n + past
    pairs = sum(min(past + i + 1, window) for i in range(n))
    return pairs, n + past - max(0, past + 1 - window)


def work(case):
    c = case
    size = 4 if c["dtype"] == "f32" else 2
    H, d = c["heads"], c["dim"]
    if c["op"] == "rotary":
        return {"bytes": c["rows"] * (2 * H * d * size + 4) + c["rot"] * 2, "flops": 3.0 * c["rows"] * H * c["rot"]}
    G, seqs = c["kv_heads"], sequences(c)
    rows = sum(n for n, _ in seqs)
    plan = sum(8 + 4 * -(-(n + past) // c["page"]) for n, past in seqs)
    if c["op"] == "append":
        return {"bytes": rows * size * (2 * H * d + 2 * G * (d + padded(d))) + plan + c["rot"] * 2, "flops": 3.0 * rows * (H + G) * c["rot"]}
    seen = [visible(n, past, c["window"]) for n, past in seqs]
    return {"bytes": 2 * rows * H * d * size + 2 * G * d * size * sum(p for _, p in seen) + plan, "flops": 4.0 * H * d * sum(p for p, _ in seen)}


# ---- in 64 bits ---------------------------------------------------------------------------------------------------------
def exact_turn(x, positions, c, f):
    """Pairs as complex numbers, multiplied by amplitude * exp(i angle)."""
    z = x.to(F64).clone()
    turn = torch.polar(torch.full((), c["amplitude"], dtype=F64, device=DEVICE), positions.to(F64)[:, None] * f.to(F64))[:, None]
    i = torch.arange(c["rot"] // 2, device=DEVICE)
    ia, ib = (i, i + c["rot"] // 2) if c["halves"] else (2 * i, 2 * i + 1)
    ia, ib = ia + c["first"], ib + c["first"]
    y = torch.complex(z[..., ia], z[..., ib]) * turn
    z[..., ia], z[..., ib] = y.real, y.imag
    return z


def exact(case, seed):
    c = case
    s = INPUTS[c["op"]](c, seed)
    d = c["dim"]
    if c["op"] == "rotary":
        x = s["x"].narrow(1, c["margin"], c["heads"] * d).reshape(c["rows"], c["heads"], d)
        return exact_turn(x, s["positions"], c, s["frequencies"])
    starts, lengths, table = (s[n].tolist() for n in ("starts", "lengths", "table"))
    if c["op"] == "append":
        H, G = c["heads"], c["kv_heads"]
        where = [(p, table[i][p // c["page"]], p % c["page"]) for i in range(len(lengths))
                 for p in range(lengths[i] - (starts[i + 1] - starts[i]), lengths[i])]
        position, page, slot = (torch.tensor(w, device=DEVICE) for w in zip(*where))
        x = s["qkv"].reshape(s["rows"], H + 2 * G, d)
        q, k = exact_turn(x[:, :H], position, c, s["frequencies"]), exact_turn(x[:, H:H + G], position, c, s["frequencies"])
        keys, values = s["keys"].to(F64), s["values"].to(F64)
        for h in range(G):
            keys[page, h, slot, :d], values[page, h, slot, :d] = k[:, h], x[:, H + G + h].to(F64)
        return [q, keys, values]
    out = torch.zeros(s["rows"], c["heads"], d, dtype=F64, device=DEVICE)
    R = c["heads"] // c["kv_heads"]
    for i, length in enumerate(lengths):
        n = starts[i + 1] - starts[i]
        all_p = torch.arange(length, device=DEVICE)
        pages = s["table"][i].long()[all_p // c["page"]]
        for h in range(c["heads"]):
            k, v = (x[pages, h // R, all_p % c["page"], :d].to(F64) for x in (s["keys"], s["values"]))
            for lo in range(0, n, 2048):
                hi = min(lo + 2048, n)
                mine = torch.arange(length - n + lo, length - n + hi, device=DEVICE)[:, None]
                ok = all_p[None] <= mine
                if c["window"]:
                    ok = ok & (mine - all_p[None] < c["window"])
                z = s["q"][starts[i] + lo:starts[i] + hi, h].to(F64) @ k.T * s["scale"]
                z = torch.where(ok, z, -math.inf)
                if s["sink"] is not None:
                    z = torch.cat([z, s["sink"][h].to(F64).expand(hi - lo, 1)], 1)
                w = torch.softmax(z, 1)[:, :length]
                out[starts[i] + lo:starts[i] + hi, h] = w @ v
    return out
