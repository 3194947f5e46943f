"""What the paged key-value cache and its attention are timed on: the write of new rows into the pages, attention over
whole prompts (packed rows, and chunks that see the pages before them), attention of single new tokens over the pages,
and the pages' own operations (free, fork, grow with copy on write, compact).

A case is a dict of plain values. prepare() makes what a serving program has in hand before the call; run() is one call
of the operator, in its plain form (elementary torch operations in float32) or, with `own`, through libosmos_amd.attn;
exact() is the same from the definition in float64, sequence by sequence.

Notation: a sequence s of a step brings the rows start[s] .. start[s + 1] - 1 and has len[s] tokens in all, these the
last; its token p lies in slot p % page of page table[s][p / page]. A cache is [layer][keys, values][page][head][slot][dim].
"""
import math
import random

import torch

own = False

TYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32, "f8": torch.float8_e4m3fn}
BYTES = {"f16": 2, "bf16": 2, "f32": 4, "f8": 1}
F8_MAX = 448.0


# ---------------------------------------------------------------- the cases

def listed():
    return [
        # a decode step of a small server: one new row for each of 48 sequences, from the projections' float rows
        dict(name="append 48 tokens f16", op="append", src="f32", cache="f16", seqs=48, rows=1, past=300, mix=1, heads=8,
             dim=128, page=16, layers=1),
        # prompts of several users going into an 8-bit cache
        dict(name="append prompts f8", op="append", src="bf16", cache="f8", seqs=7, rows=3000, past=900, mix=2, heads=4,
             dim=128, page=64, layers=2),
        # eight prompts, each sampled three ways: the last children freed, new ones forked and each grown by a token, which
        # copies the prompts' last, partly filled pages
        dict(name="fork 8 x 3, grow", op="fork", parents=8, children=3, longest=600, mix=3, heads=8, dim=128, page=16,
             layers=8, slack=64),
        # a fragmented pool made dense before it is shrunk
        dict(name="compact 6000 pages", op="compact", seqs=96, longest=1800, mix=4, heads=4, dim=128, page=16, layers=4,
             slack=3000),
        # a short question in a small model: latency
        dict(name="prompt 77 f16", op="prompt", type="f16", seqs=1, longest=77, mix=5, heads=12, kv_heads=4, dim=64,
             window=0),
        # a batch of prompts of very different lengths, packed
        dict(name="prompt 12 ragged bf16", op="prompt", type="bf16", seqs=12, longest=2111, mix=6, heads=32, kv_heads=8,
             dim=128, window=0),
        # one long prompt
        dict(name="prompt 8192 bf16", op="prompt", type="bf16", seqs=1, longest=8192, mix=7, heads=32, kv_heads=8, dim=128,
             window=0),
        # chunks of prompts that see their own earlier pages in an 8-bit cache
        dict(name="chunk 512 over f8 pages", op="chunk", type="f16", cache="f8", seqs=4, rows=512, past=6100, mix=8,
             heads=24, kv_heads=4, dim=128, page=32, layers=1, window=0),
        # one user's next token after a short prompt: latency
        dict(name="token 1 x 333 f16", op="token", type="f16", cache="f16", seqs=1, longest=333, mix=9, heads=12,
             kv_heads=4, dim=64, page=16, layers=1, window=0),
        # one user's next token in a very long context
        dict(name="token 1 x 131072 bf16", op="token", type="bf16", cache="bf16", seqs=1, longest=131072, mix=10, heads=32,
             kv_heads=8, dim=128, page=64, layers=1, window=0),
        # a serving batch of contexts of very different lengths
        dict(name="token 64 ragged bf16", op="token", type="bf16", cache="bf16", seqs=64, longest=8192, mix=11, heads=32,
             kv_heads=4, dim=128, page=16, layers=1, window=0),
        # wide heads, 8-bit pages
        dict(name="token 24 wide f8", op="token", type="bf16", cache="f8", seqs=24, longest=16384, mix=12, heads=16,
             kv_heads=2, dim=256, page=32, layers=2, window=0),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("append", "fork", "compact", "prompt", "prompt", "chunk", "token", "token"))
    mix = rng.randrange(1 << 20)
    page = rng.choice((8, 16, 32, 64, 128))
    if op == "append":
        return dict(op=op, src=rng.choice(("f32", "f16", "bf16")), cache=rng.choice(("f16", "bf16", "f8")),
                    seqs=_log(rng, 1, 64), rows=_log(rng, 1, 700), past=_log(rng, 1, 1000), mix=mix,
                    heads=rng.choice((1, 2, 4, 5, 8)), dim=rng.choice((64, 80, 96, 128, 192, 256)), page=page,
                    layers=rng.choice((1, 2)))
    if op == "fork":
        return dict(op=op, parents=_log(rng, 1, 24), children=rng.randint(1, 5), longest=_log(rng, 20, 900), mix=mix,
                    heads=rng.choice((1, 2, 4, 8)), dim=rng.choice((64, 128)), page=rng.choice((8, 16, 32, 64)),
                    layers=rng.randint(1, 8), slack=_log(rng, 130, 2000))
    if op == "compact":
        return dict(op=op, seqs=_log(rng, 2, 96), longest=_log(rng, 50, 1800), mix=mix, heads=rng.choice((1, 2, 4)),
                    dim=rng.choice((64, 128)), page=rng.choice((16, 32)), layers=rng.randint(1, 4), slack=_log(rng, 30, 3000))
    kv_heads, group = rng.choice((1, 2, 4, 8)), rng.choice((1, 2, 3, 4, 6, 8))
    while kv_heads * group > 32:
        group = rng.choice((1, 2, 3, 4))
    dim = rng.choice((64, 80, 96, 128, 128, 192, 256))
    heads = kv_heads * group
    while heads * dim > 4096:
        dim //= 2
    window = rng.choice((0, 0, 0, _log(rng, 16, 2048)))
    if op == "prompt":
        longest = _log(rng, 1, 8192)
        return dict(op=op, type=rng.choice(("f16", "bf16")), seqs=_log(rng, 1, max(1, min(24, (8192 // longest) ** 2))),
                    longest=longest, mix=mix, heads=heads, kv_heads=kv_heads, dim=dim, window=window)
    kind = rng.choice(("f16", "bf16"))
    cache = rng.choice((kind, kind, "f8"))
    if op == "chunk":
        return dict(op=op, type=kind, cache=cache, seqs=_log(rng, 1, 8), rows=_log(rng, 1, 1024), past=_log(rng, 1, 6100),
                    mix=mix, heads=heads, kv_heads=kv_heads, dim=dim, page=page, layers=rng.choice((1, 2)), window=window)
    most = min(400000, (131072 << 10) // (kv_heads * dim))
    longest = _log(rng, 1, min(131072, most))
    return dict(op=op, type=kind, cache=cache, seqs=_log(rng, 1, max(1, min(256, most // longest))), longest=longest,
                mix=mix, heads=heads, kv_heads=kv_heads, dim=dim, page=page, layers=rng.choice((1, 2)), window=window)


def _spread(mix, n, most, least=1):
    """n lengths from `least` to `most`, spread over their logarithm, the first of them `most`."""
    r = random.Random(mix)
    return [most] + [max(least, min(most, _log(r, max(1, least), most))) for _ in range(n - 1)]


def _shape(case):
    """(rows of each sequence in the step, each sequence's tokens in all)"""
    if case["op"] == "prompt":
        rows = _spread(case["mix"], case["seqs"], case["longest"])
        return rows, rows
    if case["op"] == "token":
        return [1] * case["seqs"], _spread(case["mix"], case["seqs"], case["longest"])
    rows = _spread(case["mix"], case["seqs"], case["rows"])
    past = _spread(case["mix"] + 1, case["seqs"], case["past"], 0)
    return rows, [r + p for r, p in zip(rows, past)]


def _pairs(case):
    """the (row, key) pairs that the mask leaves"""
    n = 0
    for r, m in zip(*_shape(case)):
        w = case["window"] or m
        full = min(r, max(0, m - w))  # rows that see exactly w keys: those at positions w - 1 and later
        n += full * w
        first = m - r  # the other rows see position + 1 keys
        n += sum(range(first + 1, first + 1 + r - full)) if r > full else 0
    return n


def work(case):
    op = case["op"]
    if op == "append":
        rows = sum(_shape(case)[0])
        return {"bytes": 2 * rows * case["heads"] * case["dim"] * (BYTES[case["src"]] + BYTES[case["cache"]]), "flops": 0}
    if op in ("fork", "compact"):
        page = 2 * case["layers"] * case["heads"] * case["page"] * case["dim"] * 2
        lens = _spread(case["mix"], case["parents" if op == "fork" else "seqs"], case["longest"])
        if op == "fork":
            moved = case["children"] * sum(m % case["page"] != 0 for m in lens)
            small = 8 * case["children"] * sum(-(-m // case["page"]) for m in lens)
        else:
            live = sum(-(-m // case["page"]) for m in lens)
            moved = live * case["slack"] / (live + case["slack"])
            small = 16 * live
        return {"bytes": 2 * moved * page + small, "flops": 0}
    rows, lens = _shape(case)
    q = sum(rows) * case["heads"] * case["dim"]
    seen = sum(min(m, case["window"] + r - 1) if case["window"] else m for r, m in zip(rows, lens))
    kv = seen * case["kv_heads"] * case["dim"] * 2
    return {"bytes": 2 * q * BYTES[case["type"]] + kv * BYTES[case.get("cache", case["type"])],
            "flops": 4.0 * case["heads"] * case["dim"] * _pairs(case)}


# ---------------------------------------------------------------- the inputs

def _normal(g, shape, kind, rms=1.0):
    return (torch.randn(shape, generator=g, device="cuda") * rms).to(TYPES[kind])


def _keys(g, shape, kind):
    """keys as a cache holds them: a few channels of each head much larger than the others"""
    k = torch.randn(shape, generator=g, device="cuda")
    k[..., ::29] *= 3.0
    return k.to(TYPES[kind])


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _starts(rows):
    out = [0]
    for r in rows:
        out.append(out[-1] + r)
    return out


def _pool(case, lens, g, heads, spare=0):
    """a cache with its pages dealt out in a random order, its contents and its sequences' tables"""
    page, dim, layers = case["page"], case["dim"], case["layers"]
    need = [-(-m // page) for m in lens]
    pages, width = sum(need) + spare, max(need) + 1
    order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    table = torch.full((len(lens), width), -1, dtype=torch.int32, device="cuda")
    owner = torch.repeat_interleave(torch.arange(len(lens), device="cuda"), torch.tensor(need, device="cuda"))
    first = torch.tensor(_starts(need), device="cuda")
    table[owner, torch.arange(sum(need), device="cuda") - first[owner]] = order[:sum(need)]
    return pages, table


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    op = case["op"]
    s = {"case": case}
    if op in ("fork", "compact"):
        return _prepare_pool(s, case, g)
    rows, lens = _shape(case)
    heads = case.get("kv_heads", case["heads"])
    s.update(start=_ints(_starts(rows)), len=_ints(lens), rows=max(rows), longest=max(lens), n=sum(rows))
    if op != "prompt":
        kind, layers, page, dim = case["cache"], case["layers"], case["page"], case["dim"]
        pages, s["table"] = _pool(case, lens, g, heads, 3)
        shape = (layers, pages, heads, page, dim)
        s["scale"] = None
        if kind == "f8":
            s["scale"] = 0.01 + 0.01 * torch.rand((layers, 2, heads), generator=g, device="cuda")
        data = torch.empty((layers, 2) + shape[1:], dtype=TYPES[kind], device="cuda")
        for i, made in enumerate((_keys, _normal)):
            x = made(g, shape, "f32")
            if kind == "f8":
                x = (x / s["scale"][:, i, None, :, None, None]).clamp(-F8_MAX, F8_MAX)
            data[:, i] = x.to(TYPES[kind])
        s["data"], s["layer"] = data, layers - 1
    if op == "append":
        s["k"] = _keys(g, (s["n"], heads, case["dim"]), case["src"])
        s["v"] = _normal(g, (s["n"], heads, case["dim"]), case["src"])
    else:
        shape = (s["n"], case["heads"], case["dim"])
        s["q"] = _normal(g, shape, case["type"], 1.3)
        if op == "prompt":
            s["k"] = _keys(g, (s["n"], heads, case["dim"]), case["type"])
            s["v"] = _normal(g, (s["n"], heads, case["dim"]), case["type"])
        s["soft"] = case["dim"] ** -0.5
    if own:  # the handles that a program makes once and calls every step
        from libosmos_amd import attn
        if op != "prompt":
            s["cache"] = attn.KvCache(s["data"], scale=s["scale"])
            step = attn.KvStep(s["start"], s["len"], s["table"], n_tok=s["n"], max_tok=s["rows"], max_len=s["longest"])
        if op == "append":
            s["call"] = attn.Append(s["cache"], s["layer"], step, s["k"], s["v"])
        else:
            s["out"], s["lse"] = torch.empty_like(s["q"]), torch.empty(shape[:2], device="cuda")
            if op == "prompt":
                s["call"] = attn.PromptAttention(s["q"], s["k"], s["v"], s["start"], s["rows"], s["out"], lse=s["lse"],
                                                 window=case["window"])
            else:
                kind = attn.TokenAttention if op == "token" else attn.ChunkAttention
                s["call"] = kind(s["cache"], s["layer"], step, s["q"], s["out"], lse=s["lse"], window=case["window"])
    return s


def _prepare_pool(s, case, g):
    fork = case["op"] == "fork"
    lens = _spread(case["mix"], case["parents" if fork else "seqs"], case["longest"])
    page = case["page"]
    pages, table = _pool(case, lens, g, case["heads"], case["slack"])
    seqs = len(lens) * (1 + case["children"]) if fork else len(lens)
    width = table.shape[1]
    # the counts, lengths and tables in one piece of memory
    small = torch.zeros(pages + seqs + seqs * width, dtype=torch.int32, device="cuda")
    s["small"], s["ref"], s["len"] = small, small[:pages], small[pages:pages + seqs]
    s["table"] = small[pages + seqs:].view(seqs, width)
    s["table"].fill_(-1)
    s["table"][:len(lens)] = table
    s["len"][:len(lens)] = _ints(lens)
    s["ref"][table[table >= 0].long()] = 1
    # the pages' contents, as raw words: two bytes a value
    shape = (case["layers"], 2, pages, case["heads"], page, case["dim"])
    words = torch.randint(-2 ** 31, 2 ** 31 - 1, shape[:-1] + (case["dim"] // 2,), generator=g, dtype=torch.int32,
                          device="cuda")
    s["data"] = words
    if fork:
        n, c = len(lens), case["children"]
        s["src"] = _ints([i for i in range(n) for _ in range(c)])
        s["dst"] = _ints([n + i for i in range(n * c)])
        s["grown"] = s["dst"][torch.randperm(n * c, generator=g, device="cuda")]
        s["one"] = torch.ones_like(s["dst"])
        s["done"] = torch.zeros_like(s["dst"])
    else:
        s["before"] = small.clone()
        s["live"] = torch.zeros(1, dtype=torch.int32, device="cuda")
    if own:
        from libosmos_amd import attn
        s["pool"] = attn.KvPool(attn.KvCache(words.view(torch.float16)), s["ref"], s["len"], s["table"])
    return s


# ---------------------------------------------------------------- one call

def run(s):
    op = s["case"]["op"]
    if op == "append":
        if own:
            s["call"].run()
        else:
            _append(s)
        return s["data"]
    if op == "fork":
        if own:
            s["pool"].free(s["dst"])
            s["pool"].fork(s["src"], s["dst"])
            s["pool"].grow(s["grown"], s["one"], s["done"])
        else:
            _free(s, s["dst"])
            _fork(s)
            _grow(s)
        return s["ref"], s["len"], s["table"], s["done"], s["data"]
    if op == "compact":
        s["small"].copy_(s["before"])  # the same fragmented pool for every pass: moved pages' old places keep their contents
        if own:
            s["pool"].compact(s["live"])
        else:
            _compact(s)
        return s["ref"], s["len"], s["table"], s["live"], s["data"]
    if own:
        s["call"].run()
        return s["out"], s["lse"]
    return _attend(s)


def _places(s):
    """the sequence and the position of every row of the step"""
    t = torch.arange(s["n"], device="cuda")
    start = s["start"].long()
    seq = torch.bucketize(t, start[1:], right=True)
    return t, seq, s["len"].long()[seq] - start[seq + 1] + t


def _append(s):
    case, layer = s["case"], s["layer"]
    _, seq, pos = _places(s)
    page = s["table"][seq, pos // case["page"]].long()
    slot = pos % case["page"]
    kv = torch.stack((s["k"], s["v"])).float()
    if s["scale"] is not None:
        kv = (kv / s["scale"][layer][:, None, :, None]).clamp(-F8_MAX, F8_MAX)
    kv = kv.to(TYPES[case["cache"]])
    data, kv = (s["data"].view(torch.uint8), kv.view(torch.uint8)) if s["scale"] is not None else (s["data"], kv)
    heads = torch.arange(case["heads"], device="cuda")
    data[layer, 0][page[:, None], heads, slot[:, None]] = kv[0]
    data[layer, 1][page[:, None], heads, slot[:, None]] = kv[1]


def _pages_of(s, which):
    """a layer's keys or values of every sequence in order, (sequences, heads, tokens, dim) in float32"""
    data = s["data"][s["layer"], which]
    table = s["table"].clamp(min=0).long()
    if s["scale"] is None:
        x = data[table].float()
    else:
        x = data.view(torch.uint8)[table].view(data.dtype).float() * s["scale"][s["layer"], which][:, None, None]
    b, p, h, n, d = x.shape
    return x.permute(0, 2, 1, 3, 4).reshape(b, h, p * n, d)[:, :, :s["longest"]]


def _attend(s):
    case = s["case"]
    heads, kv, dim, window = case["heads"], case["kv_heads"], case["dim"], case["window"]
    b, rows, start = s["len"].numel(), s["rows"], s["start"].long()
    n, count = s["len"].long(), (s["start"][1:] - s["start"][:-1]).long()
    at = (start[:-1, None] + torch.arange(rows, device="cuda")).clamp(max=s["n"] - 1)
    q = s["q"].float()[at].view(b, rows, kv, heads // kv, dim).permute(0, 2, 3, 1, 4).reshape(b, kv, -1, dim)
    if case["op"] == "prompt":
        k, v = (x.float()[at].permute(0, 2, 1, 3) for x in (s["k"], s["v"]))
    else:
        k, v = _pages_of(s, 0), _pages_of(s, 1)
    pos = (n - count)[:, None, None] + torch.arange(rows, device="cuda")[:, None]
    key = torch.arange(k.shape[2], device="cuda")
    seen = (key <= pos) & (key < n[:, None, None])
    if window:
        seen &= key > pos - window
    p = (q @ k.transpose(2, 3)).mul_(s["soft"]).view(b, heads, rows, -1)
    p.masked_fill_(~seen[:, None], -math.inf)
    top = p.amax(3, keepdim=True).clamp(min=-1e30)
    p = p.sub_(top).exp_()
    total = p.sum(3, keepdim=True)
    o = (p.view(b, kv, -1, p.shape[3]) @ v).view(b, heads, rows, dim) / total.clamp(min=1e-30)
    _, seq, where = _places(s)
    row = where - (n - count)[seq]
    lse = (top + total.log())[seq, :, row, 0]
    return o[seq, :, row].to(s["q"].dtype), lse


def _pages_named(s, seq):
    """(which entries of the given sequences' table rows are in use, those entries)"""
    need = -(-s["len"].long()[seq] // s["case"]["page"])
    rows = s["table"][seq]
    return torch.arange(rows.shape[1], device="cuda") < need[:, None], rows


def _count(s, pages, by):
    s["ref"].index_add_(0, pages.long(), torch.full_like(pages, by, dtype=torch.int32))


def _free(s, seq):
    seq = seq.long()
    used, rows = _pages_named(s, seq)
    _count(s, rows[used], -1)
    s["len"][seq] = 0
    s["table"][seq] = -1


def _fork(s):
    src, dst = s["src"].long(), s["dst"].long()
    used, rows = _pages_named(s, src)
    s["table"][dst] = rows
    s["len"][dst] = s["len"][src]
    _count(s, rows[used], 1)


def _grow(s):
    page, seq = s["case"]["page"], s["grown"].long()
    old = s["len"].long()[seq]
    new = old + s["one"].long()
    have, want = -(-old // page), -(-new // page)
    part = (old % page != 0) & (new > old)
    last = torch.where(part, s["table"][seq, (have - 1).clamp(min=0)].long(), -1 - torch.arange(len(seq), device="cuda"))
    before = torch.tril(last[:, None] == last, -1).sum(1)  # earlier requests for the same page: each takes a copy of its own
    copy = part & (s["ref"].long()[last.clamp(min=0)] - before > 1)
    need = want - have + copy
    free = torch.nonzero(s["ref"] == 0)[:, 0]
    ok = need.cumsum(0) <= len(free)  # in the list's order: from the first that does not fit on, all are refused
    need, copy = need * ok, copy & ok
    first = need.cumsum(0) - need
    owner = torch.repeat_interleave(torch.arange(len(seq), device="cuda"), need)
    turn = torch.arange(len(owner), device="cuda") - first[owner]
    given = free[:len(owner)]
    s["data"][:, :, given[first[copy]]] = s["data"][:, :, last[copy]]
    _count(s, last[copy], -1)
    s["table"][seq[owner], (have - copy.long())[owner] + turn] = given.to(torch.int32)
    s["ref"][given] = 1
    s["len"][seq] = torch.where(ok, new, old).to(torch.int32)
    s["done"].copy_(ok)


def _compact(s):
    ref = s["ref"]
    pages = ref.numel()
    live = ref > 0
    n = live.sum()
    ids = torch.arange(pages, device="cuda")
    hole, mover = ids[~live & (ids < n)], ids[live & (ids >= n)]
    s["data"][:, :, hole] = s["data"][:, :, mover]
    to = ids.clone()
    to[mover] = hole
    ref[hole] = ref[mover]
    ref[mover] = 0
    used, rows = _pages_named(s, torch.arange(s["len"].numel(), device="cuda"))
    s["table"].copy_(torch.where(used, to[rows.clamp(min=0).long()].to(torch.int32), rows))
    s["live"].copy_(n)


# ---------------------------------------------------------------- the same from the definition, in 64 bits

def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] in ("fork", "compact"):
        return None  # whole numbers alone
    rows, lens = _shape(case)
    if case["op"] == "append":
        layer, page = s["layer"], case["page"]
        data = s["data"].double()
        t = 0
        for i, (r, m) in enumerate(zip(rows, lens)):
            pos = torch.arange(m - r, m, device="cuda")
            at = s["table"][i].long()[pos // page]
            for j, x in enumerate((s["k"], s["v"])):
                x = x[t:t + r].double()
                if s["scale"] is not None:
                    x = x / s["scale"][layer, j].double()[:, None]
                    x = x.clamp(-F8_MAX, F8_MAX)
                data[layer, j][at, :, pos % page] = x
            t += r
        return data
    heads, group = case["heads"], case["heads"] // case["kv_heads"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    lse = torch.zeros(s["q"].shape[:2], dtype=torch.float64, device="cuda")
    t = 0
    for i, (r, m) in enumerate(zip(rows, lens)):
        pos, key = torch.arange(m - r, m, device="cuda"), torch.arange(m, device="cuda")
        dead = key > pos[:, None]
        if case["window"]:
            dead |= key <= pos[:, None] - case["window"]
        for h in range(case["kv_heads"]):
            k, v = (_exact_rows(s, case, i, h, j, t, m) for j in (0, 1))
            for a in range(h * group, (h + 1) * group):
                x = (s["q"][t:t + r, a].double() @ k.T) / math.sqrt(case["dim"])
                x[dead] = -math.inf
                z = torch.logsumexp(x, 1)
                out[t:t + r, a], lse[t:t + r, a] = torch.exp(x - z[:, None]) @ v, z
        t += r
    return out, lse


def _exact_rows(s, case, i, h, j, t, m):
    """sequence i's keys (j 0) or values (1) of head h, in float64"""
    if case["op"] == "prompt":
        return (s["k"], s["v"])[j][t:t + m, h].double()
    at = torch.arange(m, device="cuda")
    page = s["table"][i].long()[at // case["page"]]
    if s["scale"] is None:
        return s["data"][s["layer"], j][page, h, at % case["page"]].double()
    raw = s["data"].view(torch.uint8)[s["layer"], j][page, h, at % case["page"]]
    return raw.view(torch.float8_e4m3fn).double() * s["scale"][s["layer"], j, h].double()
