"""What the rows between a decoder block's products are timed on: the root-mean-square norm with the residual's addition and
the forms that the products read (mm's f16 tiles, the lane's 8-bit codes), rotary positions (over packed rows, and on the way
into the paged cache), and the choice of the next token from a row of logits.

A case is a dict of plain values. prepare() makes what a serving program has in hand before the call; run() is one call of the
operator, in its plain form (elementary torch operations in float32; angles, and sums and weights next to a rounding's or a
choice's border, in float64) or, with `own`, through libosmos_amd.rows; exact() is the same from the definition in float64.

Notation: a norm's rows are n x dim. Tiles are mm's: token t's column c at (t / 16) 16 dim + (c / 16) 256 + (t % 16) 16 + c % 16,
zeros up to a whole tile of tokens. A row's tokens are chosen from in the order of their logits, the greatest first, the lower
index first among equals. Codes are the lane's: 32 values a scale, scale = largest / 127. A rotary pair is (i, i + rot / 2)
in the half layout, (2 i, 2 i + 1) with `pairs`; what follows the first rot values of a head stays as it is. A step's rows,
lengths, tables and cache are those of perf/operators.py.
"""
import math
import random

import torch

own = False

TYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32, "f8": torch.float8_e4m3fn}
BYTES = {"f16": 2, "bf16": 2, "f32": 4, "f8": 1}
F8_MAX = 448.0
EPS = 1e-6


# ---------------------------------------------------------------- the cases

def listed():
    return [
        # one user's next token: the residual's addition and the norm before a quantised product: latency
        dict(name="norm 1 x 4096 f32 to tiles", op="norm", type="f32", add=True, to="tiles", n=1, dim=4096, pad=0),
        # a decode batch's rows on their way to the routed experts' 8-bit products
        dict(name="norm 48 x 2048 f32 to codes", op="norm", type="f32", add=True, to="codes", n=48, dim=2048, pad=0),
        # a prompt's rows of an odd width out of a wider buffer, no residual: a last norm
        dict(name="norm 700 x 4999 bf16 to rows", op="norm", type="bf16", add=False, to="f16", n=700, dim=4999, pad=9),
        # a long prompt's rows
        dict(name="norm 4096 x 6144 f32 to tiles", op="norm", type="f32", add=True, to="tiles", n=4096, dim=6144, pad=0),
        # one user's next token: its query, key and value rows, the latter two into the cache: latency
        dict(name="rope append 1 f32 to f16", op="append", type="f32", cache="f16", seqs=1, rows=1, past=777, mix=1, heads=32,
             kv_heads=8, dim=128, rot=128, pairs=False, norm=False, scaling="none", page=16),
        # a decode step of a server whose model norms its heads, rotates half of each and keeps the cache in 8 bits
        dict(name="rope append 64 normed to f8", op="append", type="f32", cache="f8", seqs=64, rows=1, past=2000, mix=2, heads=16,
             kv_heads=2, dim=256, rot=64, pairs=False, norm=True, scaling="linear", page=64),
        # prompts of several users going into a 16-bit cache, neighbouring pairs, a long context's scaling
        dict(name="rope append prompts bf16", op="append", type="bf16", cache="bf16", seqs=6, rows=1500, past=900, mix=3,
             heads=32, kv_heads=4, dim=128, rot=128, pairs=True, norm=False, scaling="bands", page=32),
        # packed rows of a long prompt's chunk, far positions, scaled
        dict(name="rope rows 8192 bf16", op="rope", type="bf16", n=8192, first=120000, heads=32, kv_heads=8, dim=128, rot=128,
             pairs=False, norm=False, scaling="yarn"),
        # one user's next token: latency
        dict(name="sample 1 x 32003 f32", op="sample", type="f32", n=1, vocab=32003, temperature=0.8, top_k=40, top_p=0.95,
             min_p=0.0, mixed=False, masked=0.0, probs=False),
        # a decode batch whose users ask for different things, a grammar's mask among them
        dict(name="sample 48 x 151001 f32 mixed", op="sample", type="f32", n=48, vocab=151001, temperature=1.0, top_k=0, top_p=1.0,
             min_p=0.0, mixed=True, masked=0.3, probs=False),
        # drafted tokens' rows, whose whole distributions are kept to accept or refuse the drafts by
        dict(name="sample 7 x 200003 f32 probs", op="sample", type="f32", n=7, vocab=200003, temperature=1.3, top_k=0, top_p=1.0,
             min_p=0.02, mixed=False, masked=0.0, probs=True),
        # the largest batch: 16-bit logits (many of them equal), a nucleus
        dict(name="sample 256 x 129024 bf16 top-p", op="sample", type="bf16", n=256, vocab=129024, temperature=1.0, top_k=0,
             top_p=0.9, min_p=0.0, mixed=False, masked=0.0, probs=False),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("norm", "norm", "rope", "append", "append", "sample", "sample"))
    if op == "norm":
        to = rng.choice(("f32", "f16", "bf16", "tiles", "tiles", "codes"))
        dim = _log(rng, 64, 8192)
        dim -= dim % {"tiles": 16, "codes": 32}.get(to, 1)
        return dict(op=op, type=rng.choice(("f32", "f32", "f16", "bf16")), add=rng.random() < 0.7, to=to, dim=dim,
                    n=_log(rng, 1, min(8192, (1 << 24) // dim)), pad=rng.choice((0, 0, 8, 9)))
    if op == "sample":
        vocab = _log(rng, 1000, 260000)
        return dict(op=op, type=rng.choice(("f32", "f32", "f16", "bf16")), n=_log(rng, 1, min(512, (1 << 24) // vocab)), vocab=vocab,
                    temperature=rng.choice((0.0, 0.7, 1.0, 1.0, rng.uniform(0.3, 1.6))), top_k=rng.choice((0, 0, 1, _log(rng, 2, vocab))),
                    top_p=rng.choice((1.0, rng.uniform(0.1, 0.99))), min_p=rng.choice((0.0, 0.0, rng.uniform(0.01, 0.3))),
                    mixed=rng.random() < 0.5, masked=rng.choice((0.0, 0.0, 0.2, 0.97)), probs=rng.random() < 0.3)
    dim = rng.choice((64, 80, 96, 128, 128, 192, 256))
    case = dict(op=op, type=rng.choice(("f32", "f16", "bf16")), dim=dim, rot=rng.choice((dim, dim, dim // 2, dim // 4)),
                kv_heads=rng.choice((1, 2, 4, 5, 8)), pairs=rng.random() < 0.4, norm=rng.random() < 0.3,
                scaling=rng.choice(("none", "none", "linear", "ntk", "yarn", "bands")))
    case["heads"] = case["kv_heads"] * rng.choice((1, 2, 3, 4))
    most = (1 << 24) // ((case["heads"] + 2 * case["kv_heads"]) * dim)
    if op == "rope":
        return dict(case, n=_log(rng, 1, min(8192, most)), first=_log(rng, 1, 1000000))
    seqs = _log(rng, 1, 64)
    return dict(case, cache=rng.choice(("f16", "bf16", "f8")), seqs=seqs, rows=rng.choice((1, _log(rng, 1, max(2, min(2000, most // seqs))))),
                past=_log(rng, 1, 2000), mix=rng.randrange(1 << 20), page=rng.choice((8, 16, 32, 64, 128)))


def _spread(mix, n, most, least=1):
    """n lengths from `least` to `most`, spread over their logarithm, the first of them `most`."""
    r = random.Random(mix)
    return [most] + [max(least, min(most, _log(r, max(1, least), most))) for _ in range(n - 1)]


def _shape(case):
    """(rows of each sequence in the step, each sequence's tokens in all)"""
    rows = _spread(case["mix"], case["seqs"], case["rows"])
    past = _spread(case["mix"] + 1, case["seqs"], case["past"], 0)
    return rows, [r + p for r, p in zip(rows, past)]


def work(case):
    op = case["op"]
    if op == "norm":
        size = BYTES[case["type"]]
        out = {"tiles": 2, "codes": 1 + 4 / 32}.get(case["to"]) or BYTES[case["to"]]
        each = size * (3 if case["add"] else 1) + out
        return {"bytes": case["n"] * case["dim"] * each + 4 * case["dim"], "flops": 5.0 * case["n"] * case["dim"]}
    if op == "sample":
        return {"bytes": case["n"] * case["vocab"] * (BYTES[case["type"]] + 4 * case["probs"]), "flops": 4.0 * case["n"] * case["vocab"]}
    size = BYTES[case["type"]]
    if op == "rope":
        values = case["n"] * (case["heads"] + case["kv_heads"]) * case["dim"]
        return {"bytes": 2 * values * size, "flops": 3.0 * values}
    rows = sum(_shape(case)[0])
    q, kv = rows * case["heads"] * case["dim"], 2 * rows * case["kv_heads"] * case["dim"]
    return {"bytes": 2 * q * size + kv * (size + BYTES[case["cache"]]), "flops": 3.0 * (q + kv / 2)}


# ---------------------------------------------------------------- the inputs

def _normal(g, shape, kind, rms=1.0):
    return (torch.randn(shape, generator=g, device="cuda") * rms).to(TYPES[kind])


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _starts(rows):
    out = [0]
    for r in rows:
        out.append(out[-1] + r)
    return out


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    s = {"case": case}
    {"norm": _prepare_norm, "sample": _prepare_sample, "rope": _prepare_rope, "append": _prepare_rope}[case["op"]](s, case, g)
    return s


def _prepare_norm(s, case, g):
    n, dim, kind = case["n"], case["dim"], case["type"]
    # a residual stream: a few channels much larger than the others
    x = torch.randn((n, dim + case["pad"]), generator=g, device="cuda")
    x[:, ::61] *= 20.0
    s["x"] = x.to(TYPES[kind])[:, :dim]
    s["add"] = _normal(g, (n, dim + case["pad"]), kind, 0.5)[:, :dim] if case["add"] else None
    s["weight"] = 1.0 + 0.2 * torch.randn(dim, generator=g, device="cuda")
    if not own:
        return
    from libosmos_amd import rows
    s["sum"] = torch.empty((n, dim), dtype=TYPES[kind], device="cuda") if case["add"] else None
    args = dict(add=s["add"], sum=s["sum"], weight=s["weight"], eps=EPS)
    if case["to"] == "tiles":
        s["out"] = torch.empty(-(-n // 16) * 16 * dim, dtype=torch.float16, device="cuda")
        s["overflow"] = torch.zeros(1, dtype=torch.int32, device="cuda")
        args.update(x16=s["out"], overflow=s["overflow"])
    elif case["to"] == "codes":
        s["codes"] = torch.empty((n, dim // 32, 32), dtype=torch.int8, device="cuda")
        s["scales"] = torch.empty((n, dim // 32, 1), device="cuda")
        args.update(codes=s["codes"], scales=s["scales"])
    else:
        s["out"] = torch.empty((n, dim), dtype=TYPES[case["to"]], device="cuda")
        args.update(out=s["out"])
    s["call"] = rows.Norm(s["x"], **args)


# a context of 4096 (8192) tokens made longer, as models state it
SCALING = {"none": None, "linear": dict(kind="linear", factor=4.0), "ntk": dict(kind="ntk", factor=8.0),
           "yarn": dict(kind="yarn", factor=16.0, context=8192, fast=32.0, slow=1.0),
           "bands": dict(kind="bands", factor=8.0, context=8192, low=1.0, high=4.0)}
BASE = 10000.0


def _prepare_rope(s, case, g):
    heads, kv, dim, kind = case["heads"], case["kv_heads"], case["dim"], case["type"]
    if case["op"] == "append":
        rows, lens = _shape(case)
        n, page = sum(rows), case["page"]
        need = [-(-m // page) for m in lens]
        pages = sum(need) + 3
        s["table"] = torch.full((len(lens), max(need)), -1, dtype=torch.int32, device="cuda")
        order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
        owner = torch.repeat_interleave(torch.arange(len(lens), device="cuda"), torch.tensor(need, device="cuda"))
        first = torch.tensor(_starts(need), device="cuda")
        s["table"][owner, torch.arange(sum(need), device="cuda") - first[owner]] = order[:sum(need)]
        s.update(start=_ints(_starts(rows)), len=_ints(lens), n=n)
        s["scale"] = 0.01 + 0.01 * torch.rand((1, 2, kv), generator=g, device="cuda") if case["cache"] == "f8" else None
        s["data"] = torch.zeros((1, 2, pages, kv, page, dim), dtype=TYPES[case["cache"]], device="cuda")
        s["v"] = _normal(g, (n, kv, dim), kind)
    else:
        n = s["n"] = case["n"]
        # packed rows of two prompts: the second begins its own positions
        pos = case["first"] + torch.arange(n, device="cuda", dtype=torch.int32)
        pos[n - n // 3:] -= case["first"] + n - n // 3
        s["pos"] = pos
    s["q"], s["k"] = _normal(g, (n, heads, dim), kind, 1.3), _normal(g, (n, kv, dim), kind)
    s["k"][..., ::29] *= 3
    s["q_weight"], s["k_weight"] = ((1.0 + 0.2 * torch.randn(dim, generator=g, device="cuda") for _ in "qk") if case["norm"] else (None, None))
    scaling = SCALING[case["scaling"]]
    if not own:  # (the table of turns a token, which a program makes once)
        s["turns"], s["factor"] = _turns(case["rot"], scaling)
        return
    from libosmos_amd import attn, rows as lib
    s["out"] = torch.empty_like(s["q"])
    turns = lib.RopeTable(case["rot"], base=BASE, scaling=scaling)
    args = dict(pairs=case["pairs"], q_weight=s["q_weight"], k_weight=s["k_weight"], eps=EPS)
    if case["op"] == "append":
        cache = attn.KvCache(s["data"], scale=s["scale"])
        step = attn.KvStep(s["start"], s["len"], s["table"], n_tok=n, max_tok=max(rows), max_len=max(lens))
        s["call"] = lib.RopeAppend(turns, cache, 0, step, s["q"], s["out"], s["k"], s["v"], **args)
    else:
        s["k_out"] = torch.empty_like(s["k"])
        s["call"] = lib.Rope(turns, s["pos"], s["q"], s["out"], s["k"], s["k_out"], **args)


def _turns(rot, scaling):
    """(turns a token of each pair in float64 on the GPU, what cosines and sines are multiplied by)"""
    base, factor = BASE, 1.0
    if scaling and scaling["kind"] == "ntk":
        base *= scaling["factor"] ** (rot / (rot - 2))
    i = torch.arange(rot // 2, dtype=torch.float64, device="cuda")
    f = base ** (-2.0 * i / rot)
    kind = scaling and scaling["kind"]
    if kind == "linear":
        f = f / scaling["factor"]
    elif kind == "yarn":
        lo, hi = (rot * math.log(scaling["context"] / (2 * math.pi * turns)) / (2 * math.log(base)) for turns in (scaling["fast"], scaling["slow"]))
        lo, hi = max(math.floor(lo), 0), min(math.ceil(hi), rot - 1)
        ramp = ((i - lo) / max(hi - lo, 0.001)).clamp(0, 1)
        f = f * (1 - ramp) + f / scaling["factor"] * ramp
        factor = 0.1 * math.log(scaling["factor"]) + 1
    elif kind == "bands":
        turns = scaling["context"] * f / (2 * math.pi)
        keep = ((turns - scaling["low"]) / (scaling["high"] - scaling["low"])).clamp(0, 1)
        f = f * keep + f / scaling["factor"] * (1 - keep)
    return f / (2 * math.pi), factor


def _prepare_sample(s, case, g):
    n, vocab = case["n"], case["vocab"]
    x = 2.5 * torch.randn((n, vocab), generator=g, device="cuda")
    # a few likely tokens a row, from a sure one to many alike
    likely = torch.randint(0, vocab, (n, 24), generator=g, device="cuda")
    x.scatter_add_(1, likely, 12.0 * torch.rand((n, 24), generator=g, device="cuda") * torch.rand((n, 1), generator=g, device="cuda"))
    if case["masked"]:
        gone = torch.rand((n, vocab), generator=g, device="cuda") < case["masked"]
        x.masked_fill_(gone, -math.inf)
        x[::2].masked_fill_(gone[::2], torch.finfo(TYPES[case["type"]]).min)
    s["logits"] = x.to(TYPES[case["type"]])
    s["u"] = torch.rand(n, generator=g, device="cuda")
    full = lambda v, t=torch.float32: torch.full((n,), v, dtype=t, device="cuda")  # noqa: E731
    s.update(temperature=full(case["temperature"]), top_k=full(case["top_k"], torch.int32), top_p=full(case["top_p"]), min_p=full(case["min_p"]))
    if case["mixed"]:  # every row asks for something of its own
        pick = torch.randint(0, 8, (4, n), generator=g, device="cuda")
        u = torch.rand((4, n), generator=g, device="cuda")
        s["temperature"] = torch.where(pick[0] == 0, 0.0, 0.3 + 1.2 * u[0])
        s["top_k"] = torch.where(pick[1] < 4, 0, (u[1] ** 4 * vocab).int() + 1).to(torch.int32)
        s["top_p"] = torch.where(pick[2] < 3, 1.0, 0.3 + 0.69 * u[2])
        s["min_p"] = torch.where(pick[3] < 5, 0.0, 0.01 + 0.2 * u[3])
    if own:
        from libosmos_amd import rows
        s["token"] = torch.empty(n, dtype=torch.int32, device="cuda")
        s["kept"] = torch.empty(n, dtype=torch.int32, device="cuda")
        s["prob"] = torch.empty(n, device="cuda")
        s["probs"] = torch.empty((n, vocab), device="cuda") if case["probs"] else None
        s["call"] = rows.Sample(s["logits"], s["u"], s["token"], temperature=s["temperature"], top_k=s["top_k"], top_p=s["top_p"],
                                min_p=s["min_p"], prob=s["prob"], kept=s["kept"], probs=s["probs"])


# ---------------------------------------------------------------- one call

def run(s):
    if not own:
        return {"norm": _norm, "rope": _rope, "append": _append, "sample": _sample}[s["case"]["op"]](s)
    s["call"].run()
    op = s["case"]["op"]
    if op == "sample":
        return (s["token"], s["prob"], s["kept"]) + ((s["probs"],) if s["case"]["probs"] else ())
    if op == "append":
        return s["out"], s["data"]
    if op == "rope":
        return s["out"], s["k_out"]
    return _normed(s, s["sum"], s["overflow"] if s["case"]["to"] == "tiles" else None,
                   s["codes"] * s["scales"] if s["case"]["to"] == "codes" else s["out"])  # (8 bits: the values they stand for)


def _normed(s, total, overflow, out):
    r = {"out": out}
    if total is not None:
        r["sum"] = total
    if overflow is not None:
        r["overflow"] = overflow
    return r


def _norm(s):
    case = s["case"]
    x = s["x"].float()
    if case["add"]:
        x = x + s["add"].float()
    if case["to"] == "codes":  # (a code's border is near: the sum as exactly as the kernels')
        r = torch.rsqrt(x.double().square().mean(1, keepdim=True) + EPS).float()
    else:
        r = torch.rsqrt(x.square().mean(1, keepdim=True) + EPS)
    y = x * r * s["weight"]
    overflow = None
    if case["to"] == "tiles":
        n, dim = y.shape
        overflow = (~(y.abs() <= 65504.0)).any().to(torch.int32).view(1)
        t = torch.zeros((-(-n // 16) * 16, dim), dtype=torch.float16, device="cuda")
        t[:n] = y
        out = t.view(-1, 16, dim // 16, 16).transpose(1, 2).reshape(-1)
    elif case["to"] == "codes":
        b = y.view(y.shape[0], -1, 32)
        top = b.abs().amax(2, keepdim=True)
        out = torch.round(b * (127.0 / top)) * (top / 127.0)
    else:
        out = y.to(TYPES[case["to"]])
    return _normed(s, x.to(s["x"].dtype) if case["add"] else None, overflow, out)


def _turned(s, x, pos, weight):
    """x (rows, heads, dim) in float32, normed where there is a weight, turned"""
    case, x = s["case"], x.float()
    rot = case["rot"]
    if weight is not None:
        x = x * torch.rsqrt(x.square().mean(2, keepdim=True) + EPS) * weight
    angle = (pos.double()[:, None] * s["turns"]) % 1.0 * (2 * math.pi)
    c, z = ((f(angle) * s["factor"]).float()[:, None] for f in (torch.cos, torch.sin))
    if case["pairs"]:
        a, b = x[..., 0:rot:2], x[..., 1:rot:2]
        y = torch.stack((a * c - b * z, b * c + a * z), 3).flatten(2)
    else:
        a, b = x[..., :rot // 2], x[..., rot // 2:rot]
        y = torch.cat((a * c - b * z, b * c + a * z), 2)
    return torch.cat((y, x[..., rot:]), 2)


def _rope(s):
    kind = s["q"].dtype
    return _turned(s, s["q"], s["pos"], s["q_weight"]).to(kind), _turned(s, s["k"], s["pos"], s["k_weight"]).to(kind)


def _append(s):
    case = s["case"]
    t, start = torch.arange(s["n"], device="cuda"), s["start"].long()
    seq = torch.bucketize(t, start[1:], right=True)
    pos = s["len"].long()[seq] - start[seq + 1] + t
    q = _turned(s, s["q"], pos, s["q_weight"]).to(s["q"].dtype)
    kv = torch.stack((_turned(s, s["k"], pos, s["k_weight"]), s["v"].float()))
    if s["scale"] is not None:
        kv = (kv / s["scale"][0][:, None, :, None]).clamp(-F8_MAX, F8_MAX)
    kv = kv.to(TYPES[case["cache"]])
    data, kv = (s["data"].view(torch.uint8), kv.view(torch.uint8)) if s["scale"] is not None else (s["data"], kv)
    page, heads = s["table"][seq, pos // case["page"]].long(), torch.arange(case["kv_heads"], device="cuda")
    for i in (0, 1):
        data[0, i][page[:, None], heads, (pos % case["page"])[:, None]] = kv[i]
    return q, s["data"]


def _sample(s):
    logits, n = s["logits"], s["case"]["vocab"]
    v, order = torch.sort(logits.float(), dim=1, descending=True, stable=True)  # (equal ones: the lowest index first)
    v = v.double()
    rank = torch.arange(n, device="cuda")
    t = s["temperature"].double()[:, None]
    greedy = ~(t > 0)
    w = torch.exp((v - v[:, :1]) / torch.where(greedy, 1.0, t))
    k = s["top_k"][:, None]
    keep = (rank < torch.where(k > 0, k, n)) & (v > -math.inf)
    w = w * keep
    c = w.cumsum(1)
    p = s["top_p"].double()[:, None]
    keep &= (c - w < p * c[:, -1:]) | (p >= 1)
    keep &= w >= s["min_p"].double()[:, None]
    keep[:, 0] = True
    keep &= ~greedy | (rank == 0)
    w = w * keep
    c = w.cumsum(1)
    total = c[:, -1:]
    at = (c <= s["u"].double()[:, None] * total).sum(1, keepdim=True)  # the first whose running sum passes u of the whole
    token, prob = order.gather(1, at), w.gather(1, at) / total
    out = token[:, 0].to(torch.int32), prob[:, 0].float(), keep.sum(1).to(torch.int32)
    return out + (torch.zeros_like(w).scatter_(1, order, w / total).float(),) if s["case"]["probs"] else out


# ---------------------------------------------------------------- the same from the definition, in 64 bits

def exact(case, seed):
    s = prepare(case, seed)
    return {"norm": _exact_norm, "rope": _exact_rope, "append": _exact_append, "sample": _exact_sample}[case["op"]](s, case)


def _exact_norm(s, case):
    total = s["x"].double() + (s["add"].double() if case["add"] else 0.0)
    y = total / torch.sqrt((total ** 2).sum(1, keepdim=True) / case["dim"] + EPS) * s["weight"].double()
    r = {"out": y}
    if case["to"] == "tiles":
        at = torch.arange(-(-case["n"] // 16) * 16 * case["dim"], device="cuda")
        tile, rest = at // (16 * case["dim"]), at % (16 * case["dim"])
        t, c = tile * 16 + rest % 256 // 16, rest // 256 * 16 + rest % 16
        r["out"] = torch.where(t < case["n"], y[t.clamp(max=case["n"] - 1), c], 0.0)
        r["overflow"] = None
    elif case["to"] == "codes":
        b = y.view(case["n"], -1, 32)
        d = b.abs().amax(2, keepdim=True) / 127
        r["out"] = torch.round(b / d) * d
    if case["add"]:
        r["sum"] = total
    return r


def _exact_turned(case, x, pos, weight):
    x, rot, scaling = x.double(), case["rot"], SCALING[case["scaling"]]
    if weight is not None:
        x = x / torch.sqrt((x ** 2).sum(2, keepdim=True) / case["dim"] + EPS) * weight.double()
    z, factor = torch.zeros((x.shape[0], rot // 2), dtype=torch.complex128, device="cuda"), 1.0
    for i in range(rot // 2):
        f = BASE ** (-2.0 * i / rot)
        if case["scaling"] == "linear":
            f /= scaling["factor"]
        elif case["scaling"] == "ntk":
            f = (BASE * scaling["factor"] ** (rot / (rot - 2))) ** (-2.0 * i / rot)
        elif case["scaling"] == "yarn":
            # the pair that makes `turns` turns in the context, as a number of pairs
            at = [rot / 2 * math.log(scaling["context"] / (2 * math.pi * turns)) / math.log(BASE) for turns in (scaling["fast"], scaling["slow"])]
            lo, hi = max(0, math.floor(at[0])), min(rot - 1, math.ceil(at[1]))
            part = min(1.0, max(0.0, (i - lo) / max(hi - lo, 0.001)))
            f = f * (1 - part) + f / scaling["factor"] * part
            factor = 1 + 0.1 * math.log(scaling["factor"])
        elif case["scaling"] == "bands":
            turns = scaling["context"] * f / (2 * math.pi)
            part = min(1.0, max(0.0, (turns - scaling["low"]) / (scaling["high"] - scaling["low"])))
            f = f * part + f / scaling["factor"] * (1 - part)
        z[:, i] = torch.polar(torch.full_like(x[:, 0, 0], factor), pos.double() * f)
    pair = (x[..., 0:rot:2], x[..., 1:rot:2]) if case["pairs"] else (x[..., :rot // 2], x[..., rot // 2:rot])
    w = torch.complex(*pair) * z[:, None]
    y = x.clone()
    if case["pairs"]:
        y[..., 0:rot:2], y[..., 1:rot:2] = w.real, w.imag
    else:
        y[..., :rot // 2], y[..., rot // 2:rot] = w.real, w.imag
    return y


def _exact_rope(s, case):
    return _exact_turned(case, s["q"], s["pos"], s["q_weight"]), _exact_turned(case, s["k"], s["pos"], s["k_weight"])


def _exact_append(s, case):
    rows, lens = _shape(case)
    pos = torch.cat([torch.arange(m - r, m, device="cuda") for r, m in zip(rows, lens)])
    q, k, v = _exact_turned(case, s["q"], pos, s["q_weight"]), _exact_turned(case, s["k"], pos, s["k_weight"]), s["v"].double()
    data, t = s["data"].double(), 0
    for i, (r, m) in enumerate(zip(rows, lens)):
        p = torch.arange(m - r, m, device="cuda")
        page = s["table"][i].long()[p // case["page"]]
        for j, x in enumerate((k, v)):
            x = x[t:t + r]
            if s["scale"] is not None:
                x = (x / s["scale"][0, j].double()[:, None]).clamp(-F8_MAX, F8_MAX)
            data[0, j][page, :, p % case["page"]] = x
        t += r
    return q, data


def _exact_sample(s, case):
    """the distributions and the drawn tokens' probabilities (the tokens and counts are whole numbers), row by row"""
    probs, all_probs = [], torch.zeros(s["logits"].shape, dtype=torch.float64, device="cuda")
    for i in range(case["n"]):
        t, k, p, m, u = (float(s[name][i]) for name in ("temperature", "top_k", "top_p", "min_p", "u"))
        l = s["logits"][i].double()
        if not t > 0:
            probs.append(1.0)
            all_probs[i, (l == l.max()).nonzero()[0, 0]] = 1.0
            continue
        kept = torch.argsort(l, descending=True, stable=True)
        kept = kept[l[kept] > -math.inf][:int(k) or None]
        w = torch.softmax(l[kept] / t, 0)
        before = torch.cat((w.new_zeros(1), w.cumsum(0)[:-1]))
        some = (w >= m * w[0]) & ((before < p) | (p >= 1))
        some[0] = True
        kept, w = kept[some], w[some] / w[some].sum()
        probs.append(float(w[int((w.cumsum(0) <= u).sum().clamp(max=len(w) - 1))]))
        all_probs[i, kept] = w
    out = None, torch.tensor(probs, dtype=torch.float64, device="cuda"), None
    return out + (all_probs,) if case["probs"] else out
