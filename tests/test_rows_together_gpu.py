"""The rows' operators as a decoder uses them (libosmos_amd.block, .rows, .layer): a small model of two blocks (norm, attention with
rotary positions over the paged cache, norm, routed experts) and its end (norm, output matrix, choice of tokens), on a prompt and then
token by token, the drawn token the next step's input. Each block against the library's single calls, bit for bit; the choice against
the definition; and the whole step captured into a graph and replayed, against the same steps queued one by one."""
import math

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
import numpy as np  # noqa: E402

from libosmos_amd import attn, capi, rows, synth  # noqa: E402
from libosmos_amd.block import AttentionLayer, TokenHead  # noqa: E402
from libosmos_amd.layer import LaneLayer  # noqa: E402

DIM, HEADS, KV, HD, PAGE, VOCAB, EXPERTS, K, FF = 512, 8, 2, 64, 16, 1040, 16, 4, 256
F32 = torch.float32


def _ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def _matrix(r, c, seed, std=0.05):
    w = np.random.default_rng(seed).normal(0, std, (r, c)).astype(np.float32)
    return synth.ID["Q4_0"], torch.from_numpy(np.ascontiguousarray(synth.quant_q4_0(w))).cuda()


def _vector(n, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return 1.0 + 0.2 * torch.randn(n, generator=g, device="cuda")


class Model:
    """two blocks and a head, with the buffers of one step of n rows"""

    def __init__(self, normed_heads):
        g = torch.Generator(device="cuda")
        g.manual_seed(77)
        self.embed = torch.randn((VOCAB, DIM), generator=g, device="cuda")
        self.cache = attn.KvCache.empty(torch.float16, 2, 60, KV, PAGE, HD)
        self.pool = attn.KvPool.empty(self.cache, 3, 20 * PAGE)
        self.rope = rows.RopeTable(HD // 2, scaling=dict(kind="yarn", factor=4.0, context=64, fast=32.0, slow=1.0))
        heads = dict(q_weight=_vector(HD, 1), k_weight=_vector(HD, 2)) if normed_heads else {}
        self.attention = [AttentionLayer(self.cache, i, HEADS, _matrix(HEADS * HD, DIM, 10 * i), _matrix(KV * HD, DIM, 10 * i + 1),
                                         _matrix(KV * HD, DIM, 10 * i + 2), _matrix(DIM, HEADS * HD, 10 * i + 3), DIM, rope=self.rope,
                                         norm=_vector(DIM, 30 + i), **heads) for i in range(2)]
        self.norms = [_vector(DIM, 40 + i) for i in range(2)]
        self.routers = [torch.randn((EXPERTS, DIM), generator=g, device="cuda").mul_(0.05) for _ in range(2)]
        t = synth.ID["Q4_0"]
        stack = lambda r, c, s: torch.stack([_matrix(r, c, s + e)[1] for e in range(EXPERTS)]).view(EXPERTS, -1)  # noqa: E731
        self.experts = [LaneLayer(t, t, DIM, FF, EXPERTS, K, stack(FF, DIM, 100), stack(FF, DIM, 200), stack(DIM, FF, 300)) for _ in range(2)]
        self.head = TokenHead(_matrix(VOCAB, DIM, 5, 0.1), VOCAB, DIM, norm=_vector(DIM, 50))

    def buffers(self, n):
        e = lambda *s, t=F32: torch.zeros(s, dtype=t, device="cuda")  # noqa: E731
        i32 = torch.int32
        return dict(x=e(n, DIM), y=e(n, DIM), h=e(n, DIM), ids=e(n, K, t=i32), w=e(n, K), zero=e(n, DIM), logits=e(n, EXPERTS), rows=e(n * K, t=i32))

    def step(self, b, calls, stream=None):
        """the blocks over b["x"] (the embedded rows), which ends as the residual stream before the last addition, b["y"]"""
        L, a, n = capi.lib(), capi.addr, b["x"].shape[0]
        add = None
        for i, layer in enumerate(self.attention):
            layer.forward(b["x"], calls[i], b["y"], stream=stream, add=add)
            # x += the attention's rows; the norm's rows to the router and the experts
            self.normed(i, b).run(stream)
            for t in range(0, n, 8):  # (mv_run takes eight rows at a time)
                assert L.mv_run(0, a(self.routers[i]), EXPERTS, DIM, a(b["h"][t:]), min(8, n - t), a(b["logits"][t:]), stream)
            assert L.q4x_route(a(b["logits"]), n, EXPERTS, K, a(b["ids"]), a(b["w"]), a(b["rows"]), stream)
            self.experts[i].forward(b["h"], b["ids"], b["w"], b["zero"], b["y"], stream)
            add = b["y"]

    def normed(self, i, b):
        key = ("norm", i)
        if key not in b:
            b[key] = rows.Norm(b["x"], add=b["y"], sum=b["x"], weight=self.norms[i], out=b["h"])
        return b[key]


def _bits(t):
    return t.contiguous().view(torch.int32)


@pytest.mark.parametrize("normed_heads", [False, True])
def test_block_is_its_calls(normed_heads):
    """AttentionLayer with a norm and rotary positions gives the bits of osmos_norm into rows, mm_x16, the products, osmos_rope,
    osmos_kv_append and the attention"""
    m, n = Model(normed_heads), 21
    other = attn.KvCache.empty(torch.float16, 2, 60, KV, PAGE, HD)
    m.pool.grow(_ints([1]), _ints([n]))
    step = attn.KvStep(_ints([0, n]), m.pool.len, m.pool.table, n_tok=n, max_tok=n, max_len=20 * PAGE, seq=_ints([1]))
    g = torch.Generator(device="cuda")
    g.manual_seed(5)
    x, add = (torch.randn((n, DIM), generator=g, device="cuda") for _ in "ab")
    out, total = torch.empty_like(x), x + add
    layer = m.attention[1]
    layer.forward(x, layer.calls(step), out, add=add)
    assert torch.equal(_bits(x), _bits(total))
    L, a = capi.lib(), capi.addr
    h = torch.empty_like(x)
    rows.Norm(total, weight=layer.norm, out=h).run()
    x16 = torch.empty((n + 15) // 16 * 16 * DIM, dtype=torch.float16, device="cuda")
    over = torch.zeros(1, dtype=torch.int32, device="cuda")
    assert L.mm_x16(a(h), DIM, n, DIM, a(x16), a(over), None)
    qkv = []
    for (t, w), r in layer.w:
        y = torch.empty((n, r // HD, HD), device="cuda")
        assert L.mm_run(t, a(w), r, DIM, a(x16), n, a(y), r, None)
        qkv.append(y)
    q, k, v = qkv
    args = dict(q_weight=layer.heads_norm["q_weight"], k_weight=layer.heads_norm["k_weight"])
    rows.Rope(m.rope, torch.arange(n, dtype=torch.int32, device="cuda"), q, q, k, k, **args).run()
    attn.Append(other, 1, step, k, v).run()
    assert torch.equal(other.data[1].view(torch.int16), m.cache.data[1].view(torch.int16))
    o = torch.zeros((n, HEADS, HD), device="cuda")
    attn.ChunkAttention(other, 1, step, q, o).run()
    o16, want = torch.empty((n + 15) // 16 * 16 * HEADS * HD, dtype=torch.float16, device="cuda"), torch.empty_like(out)
    assert L.mm_x16(a(o), HEADS * HD, n, HEADS * HD, a(o16), a(over), None)
    assert L.mm_run(layer.wo[0], a(layer.wo[1]), DIM, HEADS * HD, a(o16), n, a(want), DIM, None)
    assert torch.equal(_bits(out), _bits(want)) and torch.isfinite(out).all()


def _prompt(m, counts):
    """the prompts of len(counts) sequences, in one step; the residual stream of their last rows"""
    n = sum(counts)
    starts = [sum(counts[:i]) for i in range(len(counts) + 1)]
    m.pool.grow(_ints(range(len(counts))), _ints(counts))
    step = attn.KvStep(_ints(starts), m.pool.len, m.pool.table, n_tok=n, max_tok=max(counts), max_len=20 * PAGE)
    g = torch.Generator(device="cuda")
    g.manual_seed(6)
    b = m.buffers(n)
    tokens = torch.randint(0, VOCAB, (n,), generator=g, device="cuda", dtype=torch.int32)
    assert capi.lib().ops_gather_rows(capi.addr(b["x"]), capi.addr(m.embed), capi.addr(tokens), n, DIM, None)
    m.step(b, [layer.calls(step) for layer in m.attention])
    last = _ints([e - 1 for e in starts[1:]])
    x, y = torch.empty((len(counts), DIM), device="cuda"), torch.empty((len(counts), DIM), device="cuda")
    for dst, src in ((x, b["x"]), (y, b["y"])):
        assert capi.lib().ops_gather_rows(capi.addr(dst), capi.addr(src), capi.addr(last), len(counts), DIM, None)
    return x, y


def _limits(n):
    return dict(temperature=torch.tensor([0.0, 0.7, 1.1][:n], device="cuda"), top_k=_ints([0, 30, 0][:n]), top_p=torch.tensor([1.0, 0.9, 0.8][:n], device="cuda"))


def _defined(logits, u, limits):
    """the tokens that the definition draws, in float64"""
    out = []
    for i, l in enumerate(logits.double().cpu().numpy()):
        t, k, p, v = (float(x[i]) for x in (limits["temperature"], limits["top_k"], limits["top_p"], u))
        order = np.argsort(-l, kind="stable")
        if t == 0:
            out.append(int(order[0]))
            continue
        w = np.exp((l[order] - l[order[0]]) / t)
        w[int(k) or len(w):] = 0
        if p < 1:
            w *= np.cumsum(w) - w < p * w.sum()
        out.append(int(order[int((np.cumsum(w) <= v * w.sum()).sum())]))
    return out


def test_decoding():
    """prompts, then tokens one at a time, each drawn one the next step's input: the pages taken, the embedded rows gathered, the blocks
    and the choice queued without a wait - eagerly, and as one graph replayed"""
    counts, turns = [30, 5, 17], 6
    drawn = {}
    u = [torch.rand(3, generator=torch.Generator().manual_seed(90 + i)) for i in range(turns + 1)]
    for way in ("eager", "graph"):
        m = Model(True)
        print(way, flush=True)
        x, y = _prompt(m, counts)
        n = len(counts)
        token, v, limits = torch.zeros(n, dtype=torch.int32, device="cuda"), torch.empty(n, device="cuda"), _limits(n)
        prob, kept = torch.empty(n, device="cuda"), torch.empty(n, dtype=torch.int32, device="cuda")
        pick = m.head.calls(v, token, prob=prob, kept=kept, **limits)
        v.copy_(u[0])
        logits = m.head.forward(x, pick, add=y)
        torch.cuda.synchronize()
        assert torch.isfinite(logits).all() and float(logits.std()) > 0.1
        assert token.tolist() == _defined(logits, v, limits)
        got = [token.tolist()]
        done, seqs, one = _ints([0] * n), _ints(range(n)), _ints([1] * n)
        step = attn.KvStep(_ints(range(n + 1)), m.pool.len, m.pool.table, n_tok=n, max_tok=1, max_len=20 * PAGE, live=done)
        b, calls = m.buffers(n), [layer.calls(step) for layer in m.attention]

        def decode(stream=None):
            m.pool.grow(seqs, one, done, stream=stream)
            assert capi.lib().ops_gather_rows(capi.addr(b["x"]), capi.addr(m.embed), capi.addr(token), n, DIM, stream)
            m.step(b, calls, stream)
            m.head.forward(b["x"], pick, stream=stream, add=b["y"])

        if way == "graph":
            for i in range(2):
                m.normed(i, b)
                m.experts[i].workspace(n)
            torch.cuda.synchronize()
            graph, s = torch.cuda.CUDAGraph(), torch.cuda.Stream()
            with torch.cuda.graph(graph, stream=s):
                decode(s.cuda_stream)
        for i in range(turns):
            v.copy_(u[i + 1])
            torch.cuda.synchronize()
            if way == "graph":
                graph.replay()
            else:
                decode()
            torch.cuda.synchronize()
            assert done.tolist() == [1] * n and m.pool.len.tolist() == [c + i + 1 for c in counts]
            got.append(token.tolist())
            assert got[-1] == _defined(logits, v, limits), i
            assert (prob > 0).all() and (prob <= 1).all() and kept[0] == 1 and 1 <= int(kept[1]) <= 30
        assert not int(m.head.overflow) and not any(int(a.overflow) for a in m.attention)
        drawn[way] = got, m.cache.data.clone()
    assert drawn["eager"][0] == drawn["graph"][0]
    assert torch.equal(drawn["eager"][1].view(torch.int16), drawn["graph"][1].view(torch.int16))
    assert len({tuple(t) for t in drawn["eager"][0]}) > 2  # (the steps differ)


def test_codes_to_products():
    """the norm's codes are what the lane's products take: the bits of q8_round of its float rows"""
    n, r = 5, 64
    t, w = _matrix(r, DIM, 9)
    x, weight = torch.randn((n, DIM), generator=torch.Generator(device="cuda").manual_seed(3), device="cuda"), _vector(DIM, 3)
    out, codes, scales = torch.empty_like(x), torch.empty((n, DIM), dtype=torch.int8, device="cuda"), torch.empty((n, DIM // 32), device="cuda")
    rows.Norm(x, weight=weight, out=out, codes=codes, scales=scales).run()
    q, d = torch.empty_like(codes), torch.empty_like(scales)
    L, a = capi.lib(), capi.addr
    assert L.q8_round(a(out), n, DIM, DIM, a(q), a(d), None)
    table = torch.tensor([w.data_ptr()], dtype=torch.int64, device="cuda")
    cnt, xrow = _ints([n]), _ints([0])
    y = [torch.empty((n, r), device="cuda") for _ in "ab"]
    for (c, s), to in zip(((codes, scales), (q, d)), y):
        assert L.q8_group_tok(t, a(table), a(cnt), a(xrow), None, 1, n, r, DIM, a(c), a(s), a(to), r, None)
    assert torch.equal(_bits(y[0]), _bits(y[1])) and torch.isfinite(y[0]).all()


def test_refusals():
    m = Model(False)
    plain = AttentionLayer(m.cache, 0, HEADS, *(m.attention[0].w[i][0] for i in range(3)), m.attention[0].wo, DIM)
    m.pool.grow(_ints([0]), _ints([2]))
    step = attn.KvStep(_ints([0, 2]), m.pool.len, m.pool.table, n_tok=2, max_tok=2, max_len=20 * PAGE, seq=_ints([0]))
    x, out = torch.zeros((2, DIM), device="cuda"), torch.empty((2, DIM), device="cuda")
    with pytest.raises(ValueError):  # no norm to go with it
        plain.forward(x, plain.calls(step), out, add=x)
    with pytest.raises(ValueError):
        m.attention[0].forward(x, m.attention[0].calls(step), out, add=x[:1])
    with pytest.raises(ValueError):
        AttentionLayer(m.cache, 0, HEADS, *(m.attention[0].w[i][0] for i in range(3)), m.attention[0].wo, DIM, pairs=True)
    with pytest.raises(ValueError):
        AttentionLayer(m.cache, 0, HEADS, *(m.attention[0].w[i][0] for i in range(3)), m.attention[0].wo, DIM, rope=rows.RopeTable(128))
    with pytest.raises(TypeError):
        TokenHead(m.head.w, VOCAB, DIM, norm=torch.ones(DIM - 1, device="cuda"))
    with pytest.raises(ValueError):
        TokenHead(m.head.w, VOCAB + 1, DIM)
    token, u = _ints([0, 0]), torch.zeros(2, device="cuda")
    pick = m.head.calls(u, token)
    with pytest.raises(ValueError):
        m.head.forward(x[:1], pick)
    with pytest.raises(TypeError):
        m.head.forward(x.double(), pick)
    with pytest.raises(ValueError):
        TokenHead(m.head.w, VOCAB, DIM).forward(x, pick)
    with pytest.raises(TypeError):
        m.head.calls(u.double(), token)
    assert math.isfinite(float(m.head.forward(x, pick).abs().max()))
