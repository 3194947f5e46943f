"""Attention over packed rows and over the paged cache (osmos_attn_prompt, osmos_attn_chunk, osmos_attn_token) against a
float64 statement of it, head by head, within the error that 16-bit products with float32 sums may make: lengths from one
token on, lengths that end inside pages and tiles, sequences with no rows or fewer tokens than rows, windows, grouped
heads, every type, strided rows, tables in any order with ids out of range, and NaN in everything that is masked."""
import math

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
from tests import attn_ref  # noqa: E402

T = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32, "f8": torch.float8_e4m3fn}


def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def _starts(rows):
    out = [0]
    for r in rows:
        out.append(out[-1] + r)
    return out


def _normal(g, *shape):
    return torch.randn(shape, generator=g, device="cuda")


class Paged:
    """a cache of sequences of the given lengths: pages in a random order, NaN wherever no token lies"""

    def __init__(self, g, lens, heads, dim, page, kind, layers=2, extra=3, spread=1.0):
        from libosmos_amd import attn
        dev = "cuda"
        need = [-(-max(n, 0) // page) for n in lens]
        pages, self.width = sum(need) + extra, max(max(need), 1) + 2
        order = torch.randperm(pages, generator=g, device=dev).int()
        self.table = torch.full((len(lens), self.width), 2 ** 30, dtype=torch.int32, device=dev)  # (never to be read)
        filled = torch.zeros((pages, page), dtype=torch.bool, device=dev)
        at = 0
        for i, n in enumerate(need):
            self.table[i, :n] = order[at:at + n]
            for j in range(n):
                filled[order[at + j], :max(0, min(page, lens[i] - j * page))] = True
            at += n
        x = _normal(g, layers, 2, pages, heads, page, dim) * spread
        self.scale = None
        if kind == "f8":
            self.scale = 0.01 + 0.02 * torch.rand((layers, 2, heads), generator=g, device=dev)
            x = (x / self.scale[:, :, None, :, None, None]).clamp(-448, 448)
        x = torch.where(filled[:, None, :, None], x, math.nan)
        self.data = x.to(T[kind])
        self.len = _ints(lens)
        self.cache = attn.KvCache(self.data, self.scale)


def _case(kind, cache, heads, kv_heads, dim, page, rows, lens, window=0, q=None, out=None, seq=None, seed=0):
    return dict(kind=kind, cache=cache, heads=heads, kv_heads=kv_heads, dim=dim, page=page, rows=rows, lens=lens,
                window=window, q=q or kind, out=out or kind, seq=seq, seed=seed)


def _paged(c, token):
    from libosmos_amd import attn
    g = _gen(c["seed"])
    pg = Paged(g, c["lens"], c["kv_heads"], c["dim"], c["page"], c["cache"])
    rows, n = c["rows"], sum(c["rows"])
    seq = c["seq"] or list(range(len(rows)))
    q = (_normal(g, n, c["heads"], c["dim"]) * 1.5).to(T[c["q"]])
    out = torch.full((n, c["heads"], c["dim"]), 7.0, dtype=T[c["out"]], device="cuda")
    lse = torch.full((n, c["heads"]), 7.0, device="cuda")
    step = attn.KvStep(_ints(_starts(rows)), pg.len, pg.table, n_tok=n, max_tok=max(max(rows), 1),
                       max_len=max(max(c["lens"]), 1), seq=_ints(seq) if c["seq"] else None)
    layer = 1
    print("attn", token, c, flush=True)
    (attn.TokenAttention if token else attn.ChunkAttention)(pg.cache, layer, step, q, out, lse, window=c["window"]).run()
    torch.cuda.synchronize()
    qc = q.to(T[c["kind"]]).double()
    t = 0
    for r, s in zip(rows, seq):
        m = c["lens"][s]
        pos = torch.arange(m - r, m, device="cuda")
        for h in range(c["heads"]):
            g = h // (c["heads"] // c["kv_heads"])
            k, here = attn_ref.rows_of_pages(pg.data, pg.scale, layer, 0, pg.table[s], max(m, 0), g)
            v, _ = attn_ref.rows_of_pages(pg.data, pg.scale, layer, 1, pg.table[s], max(m, 0), g)
            want = attn_ref.attend(qc[t:t + r, h], k, v, pos, here, c["dim"] ** -0.5, c["window"], T[c["kind"]], T[c["out"]])
            attn_ref.check(out[t:t + r, h], lse[t:t + r, h], *want, (c, s, h))
        t += r


TOKEN = [
    _case("f16", "f16", 1, 1, 64, 16, [1], [1]),
    _case("f16", "f16", 8, 2, 64, 16, [1], [333]),
    _case("bf16", "bf16", 8, 1, 128, 8, [1, 1, 1, 1], [1, 17, 0, 400]),          # (a sequence of no tokens: zeros)
    _case("bf16", "bf16", 32, 8, 128, 16, [1] * 6, [1, 2, 31, 32, 33, 2500], seed=1),
    _case("f16", "f16", 3, 3, 80, 32, [1, 0, 1], [70, 50, 129]),                   # (one sequence brings no row)
    _case("f16", "f16", 24, 1, 96, 64, [1, 1], [257, 1000]),                       # (24 heads on one: more than a tile)
    _case("bf16", "bf16", 16, 2, 256, 16, [1, 1, 1], [5, 700, 64], seed=2),
    _case("f16", "f16", 2, 1, 16, 1, [1, 1], [9, 130]),                            # (pages of one token)
    _case("f16", "f16", 5, 5, 192, 128, [1, 1], [129, 640], window=100),
    _case("bf16", "bf16", 8, 2, 128, 16, [1] * 3, [3000, 40, 1025], window=1000),
    _case("bf16", "f8", 8, 2, 128, 16, [1] * 4, [1, 333, 64, 2049]),
    _case("f16", "f8", 12, 4, 80, 32, [1] * 3, [100, 31, 1500]),
    _case("f16", "f8", 4, 1, 256, 16, [1, 1], [1000, 15], window=64),
    _case("f16", "f16", 8, 2, 128, 16, [1, 1], [300, 30], q="f32", out="f32"),
    _case("bf16", "bf16", 8, 2, 64, 16, [1, 1], [300, 30], q="f32", out="f16"),
    _case("f16", "f8", 8, 2, 64, 16, [1, 1], [300, 30], q="f32", out="bf16"),
    _case("f16", "f16", 8, 2, 64, 16, [1, 1, 1], [300, 30, 70, 9], seq=[3, 0, 2]),  # (the step's sequences in another order)
    _case("bf16", "bf16", 4, 4, 128, 4096, [1, 1], [20000, 4096], seed=3),
]


@pytest.mark.parametrize("c", TOKEN, ids=range(len(TOKEN)))
def test_token(c):
    _paged(c, True)


CHUNK = [
    _case("f16", "f16", 2, 1, 64, 16, [5], [5]),
    _case("bf16", "bf16", 4, 2, 128, 16, [1, 70, 0, 130], [40, 70, 12, 500]),
    _case("f16", "f16", 6, 2, 80, 8, [33, 64], [33, 700], seed=4),
    _case("f16", "f16", 3, 1, 96, 32, [129], [1000], window=200),
    _case("bf16", "bf16", 4, 4, 192, 64, [64, 31], [64, 90]),
    _case("bf16", "bf16", 2, 1, 256, 16, [100, 260], [300, 260], seed=5),
    _case("f16", "f16", 2, 2, 16, 1, [40], [77]),
    _case("f16", "f16", 4, 1, 64, 16, [20, 30], [8, 0]),                           # (fewer tokens than rows: the first see nothing)
    _case("f16", "f8", 4, 2, 128, 32, [100, 3], [500, 3]),
    _case("bf16", "f8", 6, 1, 64, 16, [257], [1300], window=50),
    _case("f16", "f8", 2, 1, 256, 128, [65], [65]),
    _case("bf16", "f8", 3, 3, 96, 16, [80, 200], [300, 200], seed=6),
    _case("f16", "f16", 4, 2, 128, 16, [70], [300], q="f32", out="f32"),
    _case("f16", "f8", 4, 2, 128, 16, [70], [300], q="f32", out="f16"),
    _case("bf16", "bf16", 4, 2, 64, 16, [9, 70], [300, 80, 200], seq=[2, 1], out="f32"),
    _case("f16", "f16", 16, 2, 128, 16, [4, 2], [6000, 3000], seed=7),             # (few rows over long caches)
    _case("bf16", "f8", 8, 1, 256, 64, [3], [9000], seed=8),
    _case("f16", "f16", 8, 8, 64, 16, [300, 300], [2000, 300], window=1),
]


@pytest.mark.parametrize("c", CHUNK, ids=range(len(CHUNK)))
def test_chunk(c):
    _paged(c, False)


PROMPT = [
    # type, heads, kv heads, dim, rows, window, q type, out type
    ("f16", 1, 1, 64, [1], 0, "f16", "f16"),
    ("f16", 12, 4, 64, [77], 0, "f16", "f16"),
    ("bf16", 4, 1, 128, [1, 64, 0, 65, 130, 300], 0, "bf16", "bf16"),
    ("bf16", 8, 2, 128, [1100], 0, "bf16", "bf16"),
    ("f16", 3, 3, 80, [127, 33], 0, "f16", "f16"),
    ("f16", 2, 1, 96, [256, 31], 64, "f16", "f16"),
    ("bf16", 2, 2, 192, [200], 0, "bf16", "bf16"),
    ("f16", 4, 2, 256, [90, 300], 0, "f16", "f16"),
    ("f16", 2, 2, 16, [100], 7, "f16", "f16"),
    ("bf16", 2, 1, 32, [513], 300, "f32", "f32"),
    ("f16", 6, 2, 48, [129], 0, "f32", "bf16"),
    ("bf16", 10, 5, 64, [600, 20], 1, "bf16", "f16"),
    ("f16", 40, 8, 112, [150], 0, "f16", "f16"),
]


def _prompt_check(q, k, v, out, lse, rows, dim, window, kind, what):
    group = q.shape[1] // k.shape[1]
    t = 0
    for r in rows:
        pos, here = torch.arange(r, device="cuda"), torch.ones(r, dtype=torch.bool, device="cuda")
        for h in range(q.shape[1]):
            want = attn_ref.attend(q[t:t + r, h].to(T[kind]).double(), k[t:t + r, h // group].double(),
                                   v[t:t + r, h // group].double(), pos, here, dim ** -0.5, window, T[kind], out.dtype)
            attn_ref.check(out[t:t + r, h], lse[t:t + r, h], *want, (what, r, h))
        t += r


@pytest.mark.parametrize("order", ["rows", "fused", "heads"])
@pytest.mark.parametrize("c", PROMPT, ids=range(len(PROMPT)))
def test_prompt(c, order):
    """rows (tokens, heads, dim) on their own; as pieces of one fused projection; head-major tensors"""
    from libosmos_amd import attn
    kind, heads, kv, dim, rows, window, qt, ot = c
    if order != "rows" and qt != kind:
        pytest.skip("one type for all three")
    g, n = _gen(len(rows) + dim), sum(rows)
    if order == "fused":
        x = _normal(g, n, (heads + 2 * kv) * dim).to(T[kind])
        q, k, v = (x[:, a * dim:b * dim].view(n, b - a, dim) for a, b in ((0, heads), (heads, heads + kv), (heads + kv, heads + 2 * kv)))
    elif order == "heads":
        q, k, v = (_normal(g, m, n, dim).to(T[kind]).transpose(0, 1) for m in (heads, kv, kv))
    else:
        q, k, v = (_normal(g, n, m, dim).to(T[t]) for m, t in ((heads, qt), (kv, kind), (kv, kind)))
    out = torch.full((n + 1, heads, dim), 7.0, dtype=T[ot], device="cuda")
    lse = torch.zeros((n, heads), device="cuda")
    print("prompt", c, order, flush=True)
    attn.PromptAttention(q, k, v, _ints(_starts(rows)), max(rows), out[:n], lse, window=window).run()
    torch.cuda.synchronize()
    assert (out[n] == 7.0).all()
    _prompt_check(q, k, v, out[:n], lse, rows, dim, window, kind, c)


@pytest.mark.parametrize("kind", ["f16", "bf16"])
def test_large_scores(kind):
    """scores far apart and far from zero: the running maximum takes over; no overflow, no division by zero"""
    from libosmos_amd import attn
    g, n, heads, dim = _gen(5), 700, 4, 128
    q, k, v = ((_normal(g, n, heads, dim) * s).to(T[kind]) for s in (12.0, 8.0, 1.0))
    k[:, 1] -= 40.0
    q[:, 1] = q[:, 1].abs()  # (head 1: every score far below zero)
    out, lse = torch.empty_like(q), torch.empty((n, heads), device="cuda")
    print("large scores", kind, flush=True)
    attn.PromptAttention(q, k, v, _ints([0, n]), n, out, lse).run()
    torch.cuda.synchronize()
    _prompt_check(q, k, v, out, lse, [n], dim, 0, kind, "large")


@pytest.mark.parametrize("what", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("kind", ["f16", "bf16"])
def test_masked_values_have_no_influence(kind, what):
    """keys and values of NaN or infinity at token `bad`: the rows before it, and with a window those past its reach, are as
    if it were not there"""
    from libosmos_amd import attn
    g, n, heads, dim, window = _gen(6), 400, 2, 64, 90
    q, k, v = (_normal(g, n, heads, dim).to(T[kind]) for _ in range(3))
    for bad in (0, 37, 150, 399):
        for w in (0, window):
            k2, v2 = k.clone(), v.clone()
            k2[bad], v2[bad, :, ::3] = what, what
            got, lse = torch.empty_like(q), torch.empty((n, heads), device="cuda")
            print("masked", kind, what, bad, w, flush=True)
            attn.PromptAttention(q, k2, v2, _ints([0, n]), n, got, lse, window=w).run()
            torch.cuda.synchronize()
            clean = torch.arange(n, device="cuda") < bad
            if w:
                clean |= torch.arange(n, device="cuda") >= bad + w
            want, wl = torch.empty_like(q), torch.empty((n, heads), device="cuda")
            attn.PromptAttention(q, k, v, _ints([0, n]), n, want, wl, window=w).run()
            torch.cuda.synchronize()
            # (the same sums in another order at most: twice the error of one)
            tol = 2 * attn_ref.UNIT[T[kind]] * (want.double().abs() + v.double().abs().amax())
            assert ((got.double() - want.double()).abs() <= tol)[clean].all(), (bad, w)
            assert torch.allclose(lse[clean], wl[clean], rtol=1e-5, atol=1e-5)


@pytest.mark.parametrize("token", [True, False])
def test_values_alone_bad(token):
    """a value of NaN at a token that only later rows see, in the cache"""
    from libosmos_amd import attn
    g, lens = _gen(7), [100, 70]
    pg = Paged(g, lens, 2, 64, 16, "f16")
    rows = [1, 1] if token else [30, 70]
    n = sum(rows)
    q = _normal(g, n, 4, 64).half()
    step = attn.KvStep(_ints(_starts(rows)), pg.len, pg.table, n_tok=n, max_tok=max(rows), max_len=100)
    out, want = torch.empty_like(q), torch.empty_like(q)
    kind = attn.TokenAttention if token else attn.ChunkAttention
    window = 20 if token else 0
    bad = 60  # token 60: past the window of the last rows of both sequences but the second; in chunks, late
    print("values bad", token, flush=True)
    kind(pg.cache, 1, step, q, want, window=window).run()
    torch.cuda.synchronize()
    for s in (0, 1):
        pg.data[1, 1, pg.table[s, bad // 16], :, bad % 16] = math.nan
    kind(pg.cache, 1, step, q, out, window=window).run()
    torch.cuda.synchronize()
    t = 0
    for r, m in zip(rows, lens):
        for i in range(r):
            p = m - r + i
            hit = p >= bad and not (window and p - window >= bad)
            if hit:
                assert torch.isnan(out[t]).all(), p
            else:
                tol = 2.0 ** -9 * (want[t].double().abs() + 4)
                assert ((out[t].double() - want[t].double()).abs() <= tol).all(), p
            t += 1


@pytest.mark.parametrize("token", [True, False])
def test_ids_out_of_range_are_masked(token):
    """a page id below zero or past the pages: its tokens count as masked"""
    from libosmos_amd import attn
    g, lens, rows = _gen(8), [200, 64, 48], [1, 1, 1] if token else [40, 64, 10]
    pg = Paged(g, lens, 2, 64, 16, "bf16")
    pg.table[0, 3], pg.table[0, 12], pg.table[1, 0] = -1, 2 ** 31 - 1, pg.data.shape[2]
    pg.table[2, :] = -1  # (nothing of it is there)
    n = sum(rows)
    q = _normal(g, n, 4, 64).bfloat16()
    out, lse = torch.empty_like(q), torch.empty((n, 4), device="cuda")
    step = attn.KvStep(_ints(_starts(rows)), pg.len, pg.table, n_tok=n, max_tok=max(rows), max_len=200)
    print("ids", token, flush=True)
    (attn.TokenAttention if token else attn.ChunkAttention)(pg.cache, 1, step, q, out, lse).run()
    torch.cuda.synchronize()
    t = 0
    for s, (r, m) in enumerate(zip(rows, lens)):
        pos = torch.arange(m - r, m, device="cuda")
        for h in range(4):
            k, here = attn_ref.rows_of_pages(pg.data, None, 1, 0, pg.table[s], m, h // 2)
            v, _ = attn_ref.rows_of_pages(pg.data, None, 1, 1, pg.table[s], m, h // 2)
            want = attn_ref.attend(q[t:t + r, h].double(), k, v, pos, here, 0.125, 0, torch.bfloat16, torch.bfloat16)
            attn_ref.check(out[t:t + r, h], lse[t:t + r, h], *want, (s, h))
        t += r


def test_rows_outside_the_step_stay():
    """rows before the first start and from the last one on are not written"""
    from libosmos_amd import attn
    g, n = _gen(9), 100
    q, k, v = (_normal(g, n, 2, 64).half() for _ in range(3))
    out = torch.full_like(q, 7.0)
    print("outside", flush=True)
    attn.PromptAttention(q, k, v, _ints([10, 50, 50, 90]), 40, out).run()
    torch.cuda.synchronize()
    assert (out[:10] == 7.0).all() and (out[90:] == 7.0).all() and (out[10:90] != 7.0).all()


@pytest.mark.parametrize("token", [True, False])
def test_another_stream_and_graph(token):
    """on a stream of its own and captured into a graph: each replay the eager call's bits on new inputs, eager calls that
    share the workspace between the replays"""
    from libosmos_amd import attn
    import ctypes
    g, lens = _gen(10), [3000, 700, 64, 1]
    rows = [1, 1, 1, 1] if token else [5, 64, 1, 1]
    pg = Paged(g, lens, 2, 128, 16, "bf16")
    n = sum(rows)
    q = _normal(g, n, 8, 128).bfloat16()
    out, lse = torch.empty_like(q), torch.empty((n, 8), device="cuda")
    step = attn.KvStep(_ints(_starts(rows)), pg.len, pg.table, n_tok=n, max_tok=max(rows), max_len=3000)
    call = (attn.TokenAttention if token else attn.ChunkAttention)(pg.cache, 0, step, q, out, lse)
    print("graph", token, flush=True)
    call.run()
    torch.cuda.synchronize()
    s, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    with torch.cuda.stream(s):
        graph.capture_begin()
        call.run(ctypes.c_void_p(s.cuda_stream))
        graph.capture_end()
    torch.cuda.synchronize()
    for i in range(3):
        q.copy_(_normal(g, n, 8, 128))
        torch.cuda.synchronize()
        out.fill_(math.nan), lse.fill_(math.nan)
        graph.replay()
        torch.cuda.synchronize()
        a, b = out.clone(), lse.clone()
        out.fill_(math.nan)
        call.run()
        torch.cuda.synchronize()
        assert torch.isfinite(out).all() and torch.equal(a, out) and torch.equal(b, lse), i


def test_offsets_past_32_bits():
    """a cache of more than 2^32 values, its last pages read and written"""
    from libosmos_amd import attn
    page, heads, dim = 4096, 8, 256
    pages = 2 ** 32 // (page * heads * dim) + 3  # one plane past 2^32 values
    data = torch.empty((1, 2, pages, heads, page, dim), dtype=torch.float16, device="cuda")
    cache = attn.KvCache(data)
    table = _ints([[pages - 1, pages - 2]])
    n = page + 50
    g = _gen(11)
    k, v = (_normal(g, n, heads, dim).half() for _ in range(2))
    step = attn.KvStep(_ints([0, n]), _ints([n]), table, n_tok=n, max_tok=n, max_len=n)
    print("long offsets", flush=True)
    attn.Append(cache, 0, step, k, v).run()
    q = _normal(g, 1, heads, dim).half()
    out, lse = torch.empty_like(q), torch.empty((1, heads), device="cuda")
    one = attn.KvStep(_ints([0, 1]), _ints([n]), table, n_tok=1, max_tok=1, max_len=n)
    attn.TokenAttention(cache, 0, one, q, out, lse).run()
    torch.cuda.synchronize()
    o2, l2 = torch.empty_like(q), torch.empty((1, heads), device="cuda")
    attn.ChunkAttention(cache, 0, one, q, o2, l2).run()
    torch.cuda.synchronize()
    here = torch.ones(n, dtype=torch.bool, device="cuda")
    for h in range(heads):
        want = attn_ref.attend(q[:, h].double(), k[:, h].double(), v[:, h].double(), _ints([n - 1]), here, dim ** -0.5, 0,
                               torch.float16, torch.float16)
        attn_ref.check(out[:, h], lse[:, h], *want, h)
        attn_ref.check(o2[:, h], l2[:, h], *want, h)


@pytest.mark.parametrize("scale", [-0.3, 0.0, 0.5])
def test_other_scales(scale):
    """a negative scale and none: the mask and the maximum go by the scaled scores"""
    from libosmos_amd import attn
    g, lens = _gen(12), [300, 40]
    pg = Paged(g, lens, 2, 64, 16, "f16")
    here = lambda m: torch.ones(m, dtype=torch.bool, device="cuda")  # noqa: E731
    for token, rows in ((True, [1, 1]), (False, [70, 40])):
        n = sum(rows)
        q = _normal(g, n, 4, 64).half()
        out, lse = torch.empty_like(q), torch.empty((n, 4), device="cuda")
        step = attn.KvStep(_ints(_starts(rows)), pg.len, pg.table, n_tok=n, max_tok=max(rows), max_len=300)
        print("scale", scale, token, flush=True)
        (attn.TokenAttention if token else attn.ChunkAttention)(pg.cache, 1, step, q, out, lse, scale=scale).run()
        torch.cuda.synchronize()
        t = 0
        for s, (r, m) in enumerate(zip(rows, lens)):
            pos = torch.arange(m - r, m, device="cuda")
            for h in range(4):
                k, v = (attn_ref.rows_of_pages(pg.data, None, 1, w, pg.table[s], m, h // 2)[0] for w in (0, 1))
                want = list(attn_ref.attend(q[t:t + r, h].double() * math.copysign(1.0, scale), k, v, pos, here(m), abs(scale),
                                            0, torch.float16, torch.float16))
                attn_ref.check(out[t:t + r, h], lse[t:t + r, h], *want, (scale, token, s, h))
            t += r


@pytest.mark.parametrize("token", [True, False])
def test_many_sequences(token):
    """more sequences than a wave has lanes, some without rows, some without tokens; the same bits twice"""
    from libosmos_amd import attn
    g = _gen(13)
    n_seq = 150
    lens = [(37 * i * i) % 700 + (i % 3 > 0) for i in range(n_seq)]
    lens[7] = 0
    rows = [1 if i % 5 else 0 for i in range(n_seq)] if token else [min(lens[i], (11 * i) % 23) for i in range(n_seq)]
    pg = Paged(g, lens, 2, 64, 16, "bf16", layers=2)
    n = sum(rows)
    q = _normal(g, n, 4, 64).bfloat16()
    step = attn.KvStep(_ints(_starts(rows)), pg.len, pg.table, n_tok=n, max_tok=max(rows), max_len=max(lens))
    got = []
    for _ in range(2):
        out, lse = torch.full_like(q, 7.0), torch.empty((n, 4), device="cuda")
        print("many", token, flush=True)
        (attn.TokenAttention if token else attn.ChunkAttention)(pg.cache, 1, step, q, out, lse).run()
        torch.cuda.synchronize()
        got.append((out, lse))
    assert torch.equal(got[0][0], got[1][0]) and torch.equal(got[0][1], got[1][1])
    t = 0
    for s, (r, m) in enumerate(zip(rows, lens)):
        if r:
            pos = torch.arange(m - r, m, device="cuda")
            for h in (0, 3):
                (k, here), (v, _) = (attn_ref.rows_of_pages(pg.data, None, 1, w, pg.table[s], m, h // 2) for w in (0, 1))
                want = attn_ref.attend(q[t:t + r, h].double(), k, v, pos, here, 0.125, 0, torch.bfloat16, torch.bfloat16)
                attn_ref.check(out[t:t + r, h], lse[t:t + r, h], *want, (s, h))
        t += r


@pytest.mark.parametrize("kind", ["f16", "bf16"])
def test_signs_of_8_bit_scales(kind):
    """an 8-bit cache whose scales are negative or zero for some heads, and NaN among its masked bytes"""
    from libosmos_amd import attn
    g, lens = _gen(14), [500, 33, 64]
    pg = Paged(g, lens, 4, 64, 16, "f8")
    pg.scale[1, 0, 0] *= -1.0   # (keys of head 0)
    pg.scale[1, 0, 1] = 0.0     # (of head 1: every score 0)
    pg.scale[1, 1, 2] *= -1.0   # (values of head 2)
    for token, rows in ((True, [1, 1, 1]), (False, [90, 33, 5])):
        n = sum(rows)
        q = _normal(g, n, 8, 64).to(T[kind])
        out, lse = torch.empty_like(q), torch.empty((n, 8), device="cuda")
        step = attn.KvStep(_ints(_starts(rows)), pg.len, pg.table, n_tok=n, max_tok=max(rows), max_len=500)
        print("signs", kind, token, flush=True)
        (attn.TokenAttention if token else attn.ChunkAttention)(pg.cache, 1, step, q, out, lse).run()
        torch.cuda.synchronize()
        t = 0
        for s, (r, m) in enumerate(zip(rows, lens)):
            pos = torch.arange(m - r, m, device="cuda")
            for h in range(8):
                (k, here), (v, _) = (attn_ref.rows_of_pages(pg.data, pg.scale, 1, w, pg.table[s], m, h // 2) for w in (0, 1))
                want = attn_ref.attend(q[t:t + r, h].double(), k, v, pos, here, 0.125, 0, T[kind], T[kind])
                attn_ref.check(out[t:t + r, h], lse[t:t + r, h], *want, (token, s, h))
            t += r
    bad = 300  # a value's byte of NaN that only some rows of a tile see
    pg.data.view(torch.uint8)[1, 1, pg.table[0, bad // 16], :, bad % 16, ::5] = 0x7F
    rows = [220, 0, 0]
    q = _normal(g, 220, 8, 64).to(T[kind])
    out = torch.empty_like(q)
    step = attn.KvStep(_ints(_starts(rows)), pg.len, pg.table, n_tok=220, max_tok=220, max_len=500)
    attn.ChunkAttention(pg.cache, 1, step, q, out).run()
    torch.cuda.synchronize()
    sees = torch.arange(280, 500, device="cuda") >= bad
    assert torch.isnan(out[sees][..., ::5]).all() and torch.isfinite(out[~sees]).all()
    assert torch.isfinite(out[sees][..., 1::5]).all()
