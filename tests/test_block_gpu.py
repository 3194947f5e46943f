"""The attention's operators together, as a server runs them (libosmos_amd.block, .attn, .layer): a prompt's pages taken
from the pool, its rows through quantized projections into the cache and over it, the prompt forked, the children's last
page copied as they grow, each child decoded token by token, a child freed and the pool compacted in between - and the
routed experts after the attention. Each step against a float64 statement with the same roundings to f16."""
import ctypes
import math

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
import numpy as np  # noqa: E402

from tests import attn_ref  # noqa: E402

DIM, HEADS, KV, HD, PAGE = 512, 8, 2, 64, 16


def _ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def _weights(rows, cols, seed):
    from libosmos_amd import capi, synth
    w = np.random.default_rng(seed).normal(0, 0.05, (rows, cols)).astype(np.float32)
    q = torch.from_numpy(np.ascontiguousarray(synth.quant_q4_0(w))).cuda()
    f = torch.empty((rows, cols), device="cuda")
    assert capi.lib().quant_dequant(synth.ID["Q4_0"], capi.addr(q), rows * cols, capi.addr(f), None)
    torch.cuda.synchronize()
    return (synth.ID["Q4_0"], q), f.half().double()  # (mm's weights are rounded to f16)


def _half(x):
    return x.float().half().double()


class Plain:
    """the same in float64: every token's keys and values kept in order"""

    def __init__(self, wq, wk, wv, wo):
        self.wq, self.wk, self.wv, self.wo, self.k, self.v = wq, wk, wv, wo, [], []

    def fork(self):
        p = Plain(self.wq, self.wk, self.wv, self.wo)
        p.k, p.v = list(self.k), list(self.v)
        return p

    def rows(self, x):
        """(outputs, the error allowed in them) for the next rows x"""
        x = _half(x)
        q = _half(x @ self.wq.T).view(-1, HEADS, HD)
        for w, to in ((self.wk, self.k), (self.wv, self.v)):
            to.extend(_half(x @ w.T).view(-1, KV, HD))
        k, v = torch.stack(self.k), torch.stack(self.v)
        n, r = k.shape[0], q.shape[0]
        pos, here = torch.arange(n - r, n, device="cuda"), torch.ones(n, dtype=torch.bool, device="cuda")
        outs, tols = [], []
        for h in range(HEADS):
            g = h // (HEADS // KV)
            o, _, e, _ = attn_ref.attend(q[:, h], k[:, g], v[:, g], pos, here, HD ** -0.5, 0, torch.float16, torch.float32)
            # a float32 sum next to a rounding's edge may round q, k, v one f16 step (2^-10) otherwise: 2 x 2^-10 in a score's
            # products, 2^-10 in a value
            size = (q[:, h].abs() @ k[:, g].abs().T * HD ** -0.5).amax(1, keepdim=True)
            outs.append(o)
            tols.append(e + (2 * 2 * 2.0 ** -10 * size + 2.0 ** -10) * v[:, g].abs().amax())
        o, e = torch.stack(outs, 1).view(r, -1), torch.stack(tols, 1).view(r, -1)
        e = e + 2.0 ** -10 * (o.abs() + e)  # (the rounding before the output product)
        y = _half(o) @ self.wo.T
        return y, e @ self.wo.abs().T + 2.0 ** -22 * HEADS * HD * (o.abs() @ self.wo.abs().T)


def _close(got, plain, x, what):
    want, tol = plain.rows(x)
    off = (got.double() - want).abs()
    assert (off <= tol).all(), "%s: off by %.3g where %.3g is allowed" % (what, float(off.max()), float(tol.min()))
    assert (off <= 0.05 * want.abs().amax()).all(), what  # (the bound itself says something)


def test_serving_steps():
    from libosmos_amd import attn, synth
    from libosmos_amd.block import AttentionLayer
    from libosmos_amd.layer import LaneLayer
    g = torch.Generator(device="cuda")
    g.manual_seed(3)
    (wq, fq), (wk, fk), (wv, fv), (wo, fo) = (_weights(r, c, i) for i, (r, c) in enumerate(
        ((HEADS * HD, DIM), (KV * HD, DIM), (KV * HD, DIM), (DIM, HEADS * HD))))
    cache = attn.KvCache.empty(torch.float16, 2, 40, KV, PAGE, HD)
    cache.data.fill_(math.nan)  # (what no token was written to must not matter)
    pool = attn.KvPool.empty(cache, 4, 20 * PAGE)
    block = AttentionLayer(cache, 1, HEADS, wq, wk, wv, wo, DIM)
    done = _ints([0])

    def step(seqs, rows):
        n, most = sum(rows), 20 * PAGE
        starts = [sum(rows[:i]) for i in range(len(rows) + 1)]
        s = attn.KvStep(_ints(starts), pool.len, pool.table, n_tok=n, max_tok=max(rows), max_len=most, seq=_ints(seqs))
        x = torch.randn((n, DIM), generator=g, device="cuda")
        out = torch.full((n, DIM), math.nan, device="cuda")
        block.forward(x, block.calls(s), out)
        torch.cuda.synchronize()
        return x, out

    # a prompt of 77 tokens on sequence 2, in two chunks
    plain = {2: Plain(fq, fk, fv, fo)}
    for rows in (50, 27):
        pool.grow(_ints([2]), _ints([rows]), done)
        print("chunk", rows, flush=True)
        x, out = step([2], [rows])
        assert int(done) == 1
        _close(out, plain[2], x, "prompt")
    # two children of it, and all three decoded
    pool.fork(_ints([2, 2]), _ints([0, 3]))
    plain[0], plain[3] = plain[2].fork(), plain[2].fork()
    for turn in range(5):
        order = [3, 2, 0] if turn < 3 else [0, 2]
        done = _ints([0] * len(order))
        pool.grow(_ints(order), _ints([1] * len(order)), done)
        print("token", turn, flush=True)
        x, out = step(order, [1] * len(order))
        assert done.tolist() == [1] * len(order)
        for i, s in enumerate(order):
            _close(out[i:i + 1], plain[s], x[i:i + 1], ("token", turn, s))
        if turn == 2:
            pool.free(_ints([3]))
            live = _ints([0])
            pool.compact(live)
            torch.cuda.synchronize()
            used = {p for s in (0, 2) for p in pool.table[s].tolist() if p >= 0}
            assert used == set(range(int(live))) and int((pool.ref > 0).sum()) == int(live)
    # the routed experts on the attention's rows
    t3, n_exp, k, ff = synth.ID["IQ3_XXS"], 8, 2, 256
    dev = lambda a: torch.from_numpy(np.ascontiguousarray(a)).cuda()  # noqa: E731
    experts = [dev(synth.iq_blocks(t3, n_exp * r, c, 9 + i)).reshape(n_exp, -1)
               for i, (r, c) in enumerate(((ff, DIM), (ff, DIM), (DIM, ff)))]
    moe = LaneLayer(t3, t3, DIM, ff, n_exp, k, *experts)
    ids, w = _ints([[1, 5], [7, 0]]), torch.full((2, k), 0.5, device="cuda")
    y = torch.full((2, DIM), math.nan, device="cuda")
    print("experts", flush=True)
    moe.forward(out, ids, w, out, y)
    torch.cuda.synchronize()
    assert torch.isfinite(y).all()


def test_step_as_a_graph():
    """a decode step of the block captured once and replayed: each replay the eager step's bits, the append's rows too"""
    from libosmos_amd import attn
    from libosmos_amd.block import AttentionLayer
    g = torch.Generator(device="cuda")
    g.manual_seed(4)
    (wq, _), (wk, _), (wv, _), (wo, _) = (_weights(r, c, i) for i, (r, c) in enumerate(
        ((HEADS * HD, DIM), (KV * HD, DIM), (KV * HD, DIM), (DIM, HEADS * HD))))
    data = torch.randn((1, 2, 80, KV, PAGE, HD), generator=g, device="cuda").half()
    cache = attn.KvCache(data)
    pool = attn.KvPool.empty(cache, 2, 40 * PAGE)
    pool.grow(_ints([0, 1]), _ints([600, 33]))
    block = AttentionLayer(cache, 0, HEADS, wq, wk, wv, wo, DIM)
    s = attn.KvStep(_ints([0, 1, 2]), pool.len, pool.table, n_tok=2, max_tok=1, max_len=40 * PAGE)
    x, out = torch.randn((2, DIM), generator=g, device="cuda"), torch.empty((2, DIM), device="cuda")
    calls, one = block.calls(s), _ints([1, 1])
    both = _ints([0, 1])
    block.forward(x, calls, out)
    torch.cuda.synchronize()
    stream, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    at = ctypes.c_void_p(stream.cuda_stream)
    with torch.cuda.stream(stream):
        graph.capture_begin()
        pool.grow(both, one, None, at)
        block.forward(x, calls, out, at)
        graph.capture_end()
    torch.cuda.synchronize()
    for i in range(3):
        x.copy_(torch.randn((2, DIM), generator=g, device="cuda"))
        state = [t.clone() for t in (pool.ref, pool.len, pool.table, data)]
        print("replay", i, flush=True)
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in (out, pool.ref, pool.len, pool.table, data)]
        for t, was in zip((pool.ref, pool.len, pool.table, data), state):
            t.copy_(was)
        pool.grow(both, one)
        block.forward(x, calls, out)
        torch.cuda.synchronize()
        assert pool.len.tolist() == [601 + i, 34 + i]
        for a, b in zip(got, (out, pool.ref, pool.len, pool.table, data)):
            assert torch.equal(a, b), i
