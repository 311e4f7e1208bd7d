"""The paged key-value cache operators, as cases to be measured.

Four operators that a decoding engine runs beside its quantized products:

append   RoPE on the new rows' queries and keys, keys and values written to the
         cache's pages (one row per sequence in a decode step, a prompt's rows in prefill)
decode   attention of one new token per sequence over the pages
prefill  attention of a chunk of new tokens per sequence, causal, over the pages
         (the earlier positions and the chunk's own)
pages    copies of whole pages through all layers, and page tables rewritten after a
         compaction

Caches are [n_pages, n_kv_heads, page_size, head_dim] (with a leading layer axis
where all layers are meant), page tables int32 [n_seqs, pages per sequence], -1
where a sequence has no page.  Decode and prefill take a sliding window (a query
sees the last `window` positions, itself included; 0: all) and `sinks` first
positions that stay visible.

``own`` False: plain torch in 32 bits.  ``own`` True: vantablack_b200.ops.
"""
import math

import torch

own = False

DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}


# ---------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------

def _decode(name, dtype, seqs, heads, kv, hd, page, lo, hi, window=0, sinks=0):
    return dict(name=name, op="decode", dtype=dtype, seqs=seqs, heads=heads, kv=kv, hd=hd, page=page, lo=lo, hi=hi,
                window=window, sinks=sinks)


def _prefill(name, dtype, seqs, heads, kv, hd, page, q_lo, q_hi, ctx_lo, ctx_hi, window=0, sinks=0):
    return dict(name=name, op="prefill", dtype=dtype, seqs=seqs, heads=heads, kv=kv, hd=hd, page=page, q_lo=q_lo,
                q_hi=q_hi, ctx_lo=ctx_lo, ctx_hi=ctx_hi, window=window, sinks=sinks)


def _append(name, dtype, rows, seqs, heads, kv, hd, page, ctx):
    return dict(name=name, op="append", dtype=dtype, rows=rows, seqs=seqs, heads=heads, kv=kv, hd=hd, page=page,
                ctx=ctx)


def _pages(name, dtype, layers, kv, hd, page, n_pages, moves, table_seqs):
    return dict(name=name, op="pages", dtype=dtype, layers=layers, kv=kv, hd=hd, page=page, n_pages=n_pages,
                moves=moves, table_seqs=table_seqs)


def listed():
    return [
        # a single chat session early in its answer, TinyLlama's heads: latency is all
        _decode("decode-session-bf16", "bf16", 1, 32, 4, 64, 16, 37, 37),
        # the batch-32 decode of the Llama-3-8B configuration at 2048 + up to 512, in the forward loop's f32
        _decode("decode-batch32-f32", "f32", 32, 32, 8, 128, 64, 2049, 2560),
        # one reader of a very long document: the length has to be split
        _decode("decode-long-bf16", "bf16", 1, 32, 8, 128, 64, 131009, 131009),
        # streaming chats of mixed ages: sliding window with sinks, an odd group of heads
        _decode("decode-window-f16", "f16", 61, 28, 4, 128, 16, 311, 8191, 1024, 4),
        # the 2048-token prompt of the Llama-3-8B configuration
        _prefill("prefill-prompt-bf16", "bf16", 1, 32, 8, 128, 64, 2048, 2048, 0, 0),
        # a long document under a sliding window with sinks
        _prefill("prefill-window-bf16", "bf16", 1, 32, 8, 128, 64, 8192, 8192, 0, 0, 4096, 4),
        # mixed serving step: chunks of odd lengths, down to one token, over odd contexts, TinyLlama's heads
        _prefill("prefill-ragged-f16", "f16", 11, 32, 4, 64, 16, 1, 511, 3, 2049),
        # the forward loop's own type: one prefill chunk of 256 rows late in a prompt
        _prefill("prefill-chunk-f32", "f32", 1, 32, 8, 128, 64, 256, 256, 1797, 1797),
        # cache write of one batch-32 decode step, f32 cache
        _append("append-step-f32", "f32", 32, 32, 32, 8, 128, 64, 2303),
        # cache write of a long prompt, f32 rows into a bf16 cache
        _append("append-prompt-bf16", "bf16", 8191, 3, 32, 8, 128, 64, 0),
        # a TinyLlama session forked for parallel samples: a few tail pages through 22 layers
        _pages("pages-fork-f32", "f32", 22, 4, 64, 16, 64, 3, 0),
        # compaction of a fragmented Llama-3-8B cache, with the page tables of the live sequences
        _pages("pages-compact-bf16", "bf16", 32, 8, 128, 64, 256, 83, 48),
    ]


def _log(rng, lo, hi):
    """A whole number spread over the logarithm of [lo, hi]."""
    return min(hi, max(lo, int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def draw(rng):
    op = rng.choice(["decode", "decode", "prefill", "prefill", "append", "pages"])
    dtype = rng.choice(["f32", "f16", "bf16"])
    hd = rng.choice([64, 128])
    page = rng.choice([8, 16, 32, 64, 128])
    kv = rng.choice([1, 2, 3, 4, 8])
    heads = kv * rng.choice([1, 2, 3, 4, 5, 6, 7, 8, 12])
    if op == "decode":
        seqs = _log(rng, 1, 96)
        hi = _log(rng, 1, max(2, min(131072, 500000 // (seqs * kv))))
        lo = rng.randint(1, hi)
        window = rng.choice([0, 0, _log(rng, 1, 4096)])
        c = _decode("", dtype, seqs, heads, kv, hd, page, lo, hi, window, rng.choice([0, 1, 4, 5]) if window else 0)
    elif op == "prefill":
        seqs = _log(rng, 1, 12)
        most = 8192 if dtype != "f32" else 1024
        scores = 0.7e9 / (seqs * heads)  # of the plain form, which masks them: about 3 GB at most
        q_hi = _log(rng, 1, min(most // seqs, int(math.sqrt(scores))))
        q_lo = rng.randint(1, q_hi)
        room = int(scores / q_hi) - q_hi
        ctx_hi = _log(rng, 1, max(1, min(8192, room, 16384 // seqs)))
        ctx_lo = rng.randint(0, ctx_hi)
        window = rng.choice([0, 0, _log(rng, 1, 4096)])
        c = _prefill("", dtype, seqs, heads, kv, hd, page, q_lo, q_hi, ctx_lo, ctx_hi, window,
                     rng.choice([0, 1, 4, 5]) if window else 0)
    elif op == "append":
        seqs = _log(rng, 1, 64)
        c = _append("", dtype, seqs * _log(rng, 1, 8192 // seqs) - rng.randint(0, seqs - 1), seqs, heads, kv, hd, page,
                    _log(rng, 1, 2048))
    else:
        n_pages = _log(rng, 8, 256)
        layers = _log(rng, 1, 32)
        c = _pages("", dtype, layers, kv, hd, min(page, 64), n_pages, rng.randint(1, max(1, n_pages // 4)),
                   rng.choice([0, _log(rng, 1, 64)]))
    del c["name"]
    return c


# ---------------------------------------------------------------------------
# what a case's sizes come to (from the case alone, so that work() knows them)
# ---------------------------------------------------------------------------

def _spread(lo, hi, n):
    """n whole numbers from lo to hi; the seed only shuffles them."""
    return [hi] if n == 1 else [lo + (hi - lo) * i // (n - 1) for i in range(n)]


def _visible(pos, window, sinks):
    """How many positions a query at `pos` sees."""
    if not window or pos + 1 <= window:
        return pos + 1
    first = pos + 1 - window
    return window + min(sinks, first)


def _seen_by_chunk(ctx, rows, window, sinks):
    """How many cached positions the chunk [ctx, ctx + rows) sees in all."""
    first = max(0, ctx + 1 - window) if window else 0
    return ctx + rows - first + min(sinks if window else 0, first)


def work(case):
    c, es = case, SIZE[case["dtype"]]
    if c["op"] == "decode":
        seen = sum(_visible(n - 1, c["window"], c["sinks"]) for n in _spread(c["lo"], c["hi"], c["seqs"]))
        return {"bytes": es * (2 * seen * c["kv"] * c["hd"] + 2 * c["seqs"] * c["heads"] * c["hd"]),
                "flops": 4 * seen * c["heads"] * c["hd"]}
    if c["op"] == "prefill":
        seen, pairs, rows = 0, 0, 0
        for n, ctx in zip(_spread(c["q_lo"], c["q_hi"], c["seqs"]), _spread(c["ctx_lo"], c["ctx_hi"], c["seqs"])):
            seen += _seen_by_chunk(ctx, n, c["window"], c["sinks"])
            pairs += sum(_visible(p, c["window"], c["sinks"]) for p in range(ctx, ctx + n))
            rows += n
        return {"bytes": es * (2 * seen * c["kv"] * c["hd"] + 2 * rows * c["heads"] * c["hd"]),
                "flops": 4 * pairs * c["heads"] * c["hd"]}
    if c["op"] == "append":
        vals = c["rows"] * (c["heads"] + 2 * c["kv"]) * c["hd"]
        return {"bytes": vals * (4 + es) + 4 * -(-c["rows"] // c["seqs"]) * c["hd"],
                "flops": 3 * c["rows"] * (c["heads"] + c["kv"]) * c["hd"]}
    page = c["layers"] * 2 * c["kv"] * c["page"] * c["hd"] * es
    return {"bytes": 2 * c["moves"] * page + 2 * 4 * c["table_seqs"] * _table_width(c), "flops": 0}


def _table_width(c):
    return max(1, (c["n_pages"] - c["moves"]) // max(1, c["table_seqs"])) if c["table_seqs"] else 0


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------

def _table(lens, page, g, dev):
    """Pages of `lens` positions per sequence drawn from a shuffled pool: (table, number of pages)."""
    need = [-(-n // page) for n in lens]
    n_pages = sum(need) + 3
    ids = torch.randperm(n_pages, generator=g, device=dev)[: sum(need)].to(torch.int32)
    n = torch.tensor(need, device=dev)
    slot = torch.arange(max(need), device=dev)
    used = slot[None] < n[:, None]
    table = torch.full((len(lens), max(need)), -1, dtype=torch.int32, device=dev)
    table[used] = ids
    return table, n_pages


def _shuffle(values, g, dev):
    at = torch.randperm(len(values), generator=g, device=dev).tolist()
    return [values[i] for i in at]


def prepare(case, seed):
    c, dev = case, torch.device("cuda")
    g = torch.Generator(device=dev)
    g.manual_seed(int(seed))
    dt = DT[c["dtype"]]

    def normal(*shape, dtype=dt):
        return torch.randn(*shape, generator=g, device=dev, dtype=torch.float32).to(dtype)

    s = {"case": dict(c)}
    if c["op"] in ("decode", "prefill"):
        if c["op"] == "decode":
            lens = _shuffle(_spread(c["lo"], c["hi"], c["seqs"]), g, dev)
            rows = c["seqs"]
        else:
            qn = _spread(c["q_lo"], c["q_hi"], c["seqs"])
            cx = _spread(c["ctx_lo"], c["ctx_hi"], c["seqs"])
            both = _shuffle(list(zip(qn, cx)), g, dev)
            lens = [a + b for a, b in both]
            rows = sum(qn)
            starts = [0]
            for a, _ in both:
                starts.append(starts[-1] + a)
            s["starts"] = torch.tensor(starts, dtype=torch.int32, device=dev)
            s["q_max"] = max(qn)
        s["table"], n_pages = _table(lens, c["page"], g, dev)
        s["lens"] = torch.tensor(lens, dtype=torch.int32, device=dev)
        s["k"] = normal(n_pages, c["kv"], c["page"], c["hd"])
        s["v"] = normal(n_pages, c["kv"], c["page"], c["hd"])
        s["q"] = normal(rows, c["heads"], c["hd"])
        s["scale"] = 1.0 / math.sqrt(c["hd"])
    elif c["op"] == "append":
        rows, seqs = c["rows"], c["seqs"]
        per = -(-rows // seqs)
        count = [min(per, max(0, rows - i * per)) for i in range(seqs)]
        s["table"], n_pages = _table([c["ctx"] + per] * seqs, c["page"], g, dev)
        s["seq"] = torch.arange(rows, device=dev, dtype=torch.int32) // per
        s["pos"] = (torch.arange(rows, device=dev, dtype=torch.int32) % per) + c["ctx"]
        s["k"] = normal(n_pages, c["kv"], c["page"], c["hd"])
        s["v"] = normal(n_pages, c["kv"], c["page"], c["hd"])
        # one projection's output, Q | K | V side by side, as the forward loop leaves it
        s["qkv"] = normal(rows, (c["heads"] + 2 * c["kv"]) * c["hd"], dtype=torch.float32)
        s["q_out"] = torch.zeros(rows, c["heads"], c["hd"], dtype=dt, device=dev)
        inv = 1.0 / (500000.0 ** (torch.arange(0, c["hd"], 2, device=dev, dtype=torch.float64) / c["hd"]))
        ang = torch.arange(c["ctx"] + max(count), device=dev, dtype=torch.float64)[:, None] * inv
        # [position, head_dim]: (cos, sin) of each rotated pair
        s["rope"] = torch.stack((ang.cos(), ang.sin()), -1).reshape(ang.shape[0], c["hd"]).float()
    else:
        shape = (c["layers"], c["n_pages"], c["kv"], c["page"], c["hd"])
        s["k"], s["v"] = normal(*shape), normal(*shape)
        # live pages lie anywhere; the moves take the live pages behind the first n - moves
        # places into the holes before them (distinct sources, distinct targets, none both)
        keep = c["n_pages"] - c["moves"]
        order = torch.randperm(keep, generator=g, device=dev)
        s["dst"] = order[: c["moves"]].to(torch.int32)
        s["src"] = (keep + torch.randperm(c["moves"], generator=g, device=dev)).to(torch.int32)
        if c["table_seqs"]:
            s["map"] = torch.arange(c["n_pages"], device=dev, dtype=torch.int32)
            s["map"][s["src"].long()] = s["dst"]
            live = torch.cat((order[c["moves"]:].to(torch.int32), s["src"]))
            live = live[torch.randperm(live.numel(), generator=g, device=dev)]
            w = _table_width(c)
            table = torch.full((c["table_seqs"] * w,), -1, dtype=torch.int32, device=dev)
            n = min(live.numel(), table.numel())
            table[:n] = live[:n]
            s["table"] = table.view(c["table_seqs"], w)
    return s


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------

def run(state):
    s, c = state, state["case"]
    if own:
        from vantablack_b200 import ops
        if c["op"] == "decode":
            return ops.paged_attention_decode(s["q"], s["k"], s["v"], s["table"], s["lens"], scale=s["scale"],
                                              window=c["window"], sinks=c["sinks"])
        if c["op"] == "prefill":
            return ops.paged_attention_prefill(s["q"], s["k"], s["v"], s["table"], s["lens"], s["starts"],
                                               scale=s["scale"], window=c["window"], sinks=c["sinks"])
        if c["op"] == "append":
            h, n, hd = c["heads"], c["kv"], c["hd"]
            rows = s["qkv"].view(c["rows"], h + 2 * n, hd)
            ops.paged_append(s["k"], s["v"], s["table"], rows[:, h:h + n], rows[:, h + n:], s["seq"], s["pos"],
                             q=rows[:, :h], q_out=s["q_out"], rope=s["rope"])
            return s["q_out"], s["k"], s["v"]
        ops.paged_copy(s["k"], s["v"], s["src"], s["dst"], page_table=s.get("table"), page_map=s.get("map"))
        return (s["k"], s["v"], s["table"]) if "table" in s else (s["k"], s["v"])
    if c["op"] == "decode":
        return _plain_attention(s, s["q"][:, None], s["lens"][:, None].long() - 1)[:, 0]
    if c["op"] == "prefill":
        n = s["starts"][1:] - s["starts"][:-1]
        at = torch.arange(s["q_max"], device=n.device)
        row = (s["starts"][:-1, None] + at).clamp(max=s["q"].shape[0] - 1).long()
        pos = (s["lens"] - n)[:, None] + at
        out = _plain_attention(s, s["q"][row], pos.long())
        # back to the packed rows: row r belongs to the sequence whose start is the last one not behind it
        r = torch.arange(s["q"].shape[0], device=n.device, dtype=torch.int32)
        seq = torch.searchsorted(s["starts"], r, right=True) - 1
        return out[seq, r - s["starts"][seq]]
    if c["op"] == "append":
        return _plain_append(s)
    s["k"][:, s["dst"].long()] = s["k"][:, s["src"].long()]
    s["v"][:, s["dst"].long()] = s["v"][:, s["src"].long()]
    if "table" not in s:
        return s["k"], s["v"]
    t = s["table"]
    t.copy_(torch.where(t >= 0, s["map"][t.clamp(min=0).long()], t))
    return s["k"], s["v"], t


def _plain_attention(s, q, pos):
    """q [seqs, rows, heads, hd] at positions pos [seqs, rows] over each sequence's pages, in 32 bits."""
    c = s["case"]
    b, rows, heads, hd = q.shape
    kv, group = c["kv"], heads // c["kv"]
    ids = s["table"].clamp(min=0).long()
    length = ids.shape[1] * c["page"]
    k = s["k"][ids].transpose(1, 2).reshape(b, kv, length, hd).float()
    v = s["v"][ids].transpose(1, 2).reshape(b, kv, length, hd).float()
    t = torch.arange(length, device=q.device)
    see = (t <= pos[..., None]) & (t < s["lens"][:, None, None])
    if c["window"]:
        see &= (t > pos[..., None] - c["window"]) | (t < c["sinks"])
    qs = q.view(b, rows, kv, group, hd).permute(0, 2, 1, 3, 4).reshape(b, kv, rows * group, hd).float() * s["scale"]
    x = qs @ k.transpose(-1, -2)
    x = x.view(b, kv, rows, group, length).masked_fill_(~see[:, None, :, None], -math.inf)
    m = x.amax(-1, keepdim=True)
    p = x.sub_(torch.where(m == -math.inf, 0.0, m)).exp_()
    l = p.sum(-1, keepdim=True)
    o = (p.view(b, kv, rows * group, length) @ v).view(b, kv, rows, group, hd)
    o = torch.where(l > 0, o / l, 0.0)
    return o.permute(0, 2, 1, 3, 4).reshape(b, rows, heads, hd).to(q.dtype)


def _plain_append(s):
    c = s["case"]
    h, n, hd, dt = c["heads"], c["kv"], c["hd"], s["k"].dtype
    x = s["qkv"].view(c["rows"], h + 2 * n, hd)
    cs = s["rope"][s["pos"].long()].view(c["rows"], 1, hd // 2, 2)
    a = x[:, : h + n].reshape(c["rows"], h + n, hd // 2, 2)
    y = torch.stack((a[..., 0] * cs[..., 0] - a[..., 1] * cs[..., 1], a[..., 0] * cs[..., 1] + a[..., 1] * cs[..., 0]), -1)
    y = y.reshape(c["rows"], h + n, hd).to(dt)
    page = s["table"][s["seq"].long(), s["pos"].long() // c["page"]].long()
    slot = s["pos"].long() % c["page"]
    s["q_out"].copy_(y[:, :h])
    s["k"][page, :, slot] = y[:, h:]
    s["v"][page, :, slot] = x[:, h + n:].to(dt)
    return s["q_out"], s["k"], s["v"]


# ---------------------------------------------------------------------------
# the definition, in 64 bits
# ---------------------------------------------------------------------------

def exact(case, seed):
    s, c = prepare(case, seed), case
    if c["op"] == "decode":
        lens = s["lens"].tolist()
        return torch.stack([_exact_rows(s, s["q"][i:i + 1], i, n - 1, n)[0] for i, n in enumerate(lens)])
    if c["op"] == "prefill":
        lens, starts = s["lens"].tolist(), s["starts"].tolist()
        out = [_exact_rows(s, s["q"][a:b], i, lens[i] - (b - a), lens[i])
               for i, (a, b) in enumerate(zip(starts, starts[1:]))]
        return torch.cat(out)
    if c["op"] == "append":
        h, n, hd = c["heads"], c["kv"], c["hd"]
        x = s["qkv"].double().view(c["rows"], h + 2 * n, hd)
        z = torch.view_as_complex(x[:, : h + n].reshape(c["rows"], h + n, hd // 2, 2).contiguous())
        turn = torch.view_as_complex(s["rope"].double().view(-1, hd // 2, 2).contiguous())
        y = torch.view_as_real(z * turn[s["pos"].long()][:, None]).reshape(c["rows"], h + n, hd)
        k, v = s["k"].double(), s["v"].double()
        flat = s["table"][s["seq"].long(), torch.div(s["pos"], c["page"], rounding_mode="floor").long()].long()
        for head in range(n):
            k[flat, head, s["pos"].long() % c["page"]] = y[:, h + head]
            v[flat, head, s["pos"].long() % c["page"]] = x[:, h + n + head]
        return y[:, :h].contiguous(), k, v
    k, v = s["k"].clone(), s["v"].clone()  # moved bits: nothing is rounded
    for a, b in zip(s["src"].tolist(), s["dst"].tolist()):
        k[:, b], v[:, b] = s["k"][:, a], s["v"][:, a]
    return (k.double(), v.double(), None) if "table" in s else (k.double(), v.double())


def _exact_rows(s, q, seq, first, length):
    """Rows of one sequence at positions first, first + 1, ...: softmax(scale q k^T) v over what each sees."""
    c = s["case"]
    rows, heads, hd = q.shape
    group = heads // c["kv"]
    t = torch.arange(length, device=q.device)
    page = s["table"][seq].long()[torch.div(t, c["page"], rounding_mode="floor")]
    hidden = t[None] > (first + torch.arange(rows, device=q.device))[:, None]
    if c["window"]:
        pos = (first + torch.arange(rows, device=q.device))[:, None]
        hidden |= (pos - t[None] >= c["window"]) & (t[None] >= c["sinks"])
    out = torch.empty(rows, heads, hd, dtype=torch.float64, device=q.device)
    for n in range(c["kv"]):
        k, v = s["k"][page, n, t % c["page"]].double(), s["v"][page, n, t % c["page"]].double()
        for j in range(n * group, (n + 1) * group):
            x = (q[:, j].double() @ k.T) * s["scale"]
            out[:, j] = torch.softmax(x.masked_fill_(hidden, -math.inf), -1) @ v
    return out
