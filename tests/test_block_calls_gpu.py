"""AttentionLayer's steps and their buffers (libosmos_amd.block): a step runs on the rows and buffers that its calls were made for."""
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

from tests.test_block_gpu import DIM, HD, HEADS, KV, PAGE, _ints, _weights  # noqa: E402


def _layer(pages=60, seqs=2):
    from libosmos_amd import attn
    from libosmos_amd.block import AttentionLayer
    w = [_weights(r, c, i)[0] for i, (r, c) in enumerate(((HEADS * HD, DIM), (KV * HD, DIM), (KV * HD, DIM), (DIM, HEADS * HD)))]
    cache = attn.KvCache.empty(torch.float16, 1, pages, KV, PAGE, HD)
    pool = attn.KvPool.empty(cache, seqs, 40 * PAGE)
    return cache, pool, AttentionLayer(cache, 0, HEADS, *w, DIM)


def _step(pool, rows):
    from libosmos_amd import attn
    starts = [sum(rows[:i]) for i in range(len(rows) + 1)]
    return attn.KvStep(_ints(starts), pool.len, pool.table, n_tok=sum(rows), max_tok=max(rows), max_len=40 * PAGE)


def test_rows_of_another_step_are_refused():
    cache, pool, layer = _layer()
    pool.grow(_ints([0, 1]), _ints([3, 1]))
    calls = layer.calls(_step(pool, [3, 1]))
    layer.calls(_step(pool, [1, 1]))
    x, out = (torch.zeros((4, DIM), device="cuda") for _ in range(2))
    torch.cuda.synchronize()
    before = cache.data.clone()
    wide = torch.zeros((4, 2 * DIM), device="cuda")
    bad = [(x[:2], out[:2]), (x[:2], out), (x, out[:3]), (x.half(), out), (x, out.half()), (x.double(), out), (wide[:, :DIM], out),
           (x, wide[:, :DIM]), (x.T.contiguous().T, out), (x.cpu(), out), (x.view(2, 2 * DIM), out), (x.view(-1), out)]
    for a, b in bad:
        print("refused", tuple(a.shape), a.dtype, tuple(b.shape), b.dtype, flush=True)
        with pytest.raises((TypeError, ValueError)):
            layer.forward(a, calls, b)
    other = _layer()[2]
    with pytest.raises(ValueError):
        other.forward(x, calls, out)
    torch.cuda.synchronize()
    assert torch.equal(cache.data, before)
    layer.forward(x, calls, out)
    torch.cuda.synchronize()
    assert (out == 0).all()


def test_overflow_is_reported():
    """layer.overflow: 0 while every row fits f16, 1 once one does not, until the caller clears it"""
    cache, pool, layer = _layer()
    pool.grow(_ints([0, 1]), _ints([2, 2]))
    calls = layer.calls(_step(pool, [2, 2]))
    out = torch.empty((4, DIM), device="cuda")
    for value, want in ((1.0, 0), (65504.0, 0), (65510.0, 1), (1.0, 1)):
        x = torch.zeros((4, DIM), device="cuda")
        x[2, 7] = value
        layer.forward(x, calls, out)
        torch.cuda.synchronize()
        assert layer.overflow.tolist() == [want], value
    layer.overflow.zero_()
    layer.forward(x, calls, out)
    torch.cuda.synchronize()
    assert layer.overflow.tolist() == [0]


def test_rows_of_no_sequence_stay_finite():
    """rows that a step's sequences leave out (a batch padded to one size) reach neither the cache nor the overflow flag"""
    from libosmos_amd import attn
    cache, pool, layer = _layer()
    pool.grow(_ints([0, 1]), _ints([1, 1]))
    junk = torch.full((1 << 20,), float("inf"), device="cuda")  # (what new buffers may be made of)
    del junk
    step = attn.KvStep(_ints([0, 1, 2]), pool.len, pool.table, n_tok=16, max_tok=1, max_len=40 * PAGE)
    x, out = torch.randn((16, DIM), device="cuda"), torch.empty((16, DIM), device="cuda")
    layer.forward(x, layer.calls(step), out)
    torch.cuda.synchronize()
    assert layer.overflow.tolist() == [0] and torch.isfinite(out).all()


def test_one_set_of_buffers():
    """prompts of many lengths: the layer keeps the buffers of the longest, and calls made before and after it run right on their own"""
    cache, pool, layer = _layer(pages=200, seqs=1)
    pool.grow(_ints([0]), _ints([640]))
    cache.data.copy_(torch.randn(cache.data.shape, device="cuda"))
    a_row = (HEADS + 2 * KV + HEADS) * HD * 4 + (DIM + HEADS * HD) * 2
    first, outs = layer.calls(_step(pool, [3])), {}
    x = torch.randn((640, DIM), device="cuda")
    torch.cuda.synchronize()
    start = torch.cuda.memory_allocated()
    for n in range(1, 641, 9):
        layer.calls(_step(pool, [n]))
    kept = torch.cuda.memory_allocated() - start
    assert kept <= 1.1 * 656 * a_row + (1 << 20), "%d bytes kept where one set of 640 rows is %d" % (kept, 640 * a_row)

    def run(calls, n):
        out = torch.full((n, DIM), float("nan"), device="cuda")
        layer.forward(x[:n], calls, out)
        torch.cuda.synchronize()
        return out
    late = {n: layer.calls(_step(pool, [n])) for n in (3, 640, 17)}
    alone = {n: _layer_like(layer, cache) for n in (3, 640, 17)}
    for n in (3, 640, 17, 3):
        other = torch.full((n, DIM), float("nan"), device="cuda")
        alone[n].forward(x[:n], alone[n].calls(_step(pool, [n])), other)
        torch.cuda.synchronize()
        outs[n] = other
        assert torch.equal(run(late[n], n), other), n
    alone[3].forward(x[:3], alone[3].calls(_step(pool, [3])), outs[3])  # (the tokens of the last step again)
    torch.cuda.synchronize()
    assert torch.equal(run(first, 3), outs[3])


def _layer_like(layer, cache):
    from libosmos_amd.block import AttentionLayer
    return AttentionLayer(cache, 0, HEADS, *[w for w, _ in layer.w], layer.wo, DIM)


def _rotate(x, pos):
    """rotary positions: pairs (i, i + HD / 2) turned by pos 10000^(-2 i / HD), in place"""
    half = x.shape[-1] // 2
    angle = pos[:, None].double() * 10000.0 ** (-2.0 * torch.arange(half, device="cuda").double() / x.shape[-1])
    c, s = angle.cos()[:, None].to(x.dtype), angle.sin()[:, None].to(x.dtype)
    a, b = x[..., :half].clone(), x[..., half:].clone()
    x[..., :half], x[..., half:] = a * c - b * s, a * s + b * c


@pytest.mark.parametrize("rows", [1, 40])
def test_positions_between_projections_and_cache(rows):
    """a step with rotary positions on its queries and keys: the cache holds the turned keys, and the outputs are those of the same
    rows turned and attended call by call"""
    from libosmos_amd import attn
    cache, pool, layer = _layer(seqs=2)
    cache.data.copy_(torch.randn(cache.data.shape, device="cuda"))
    pool.grow(_ints([0, 1]), _ints([77, 300]))
    step = _step(pool, [rows, rows])
    n = 2 * rows
    pos = torch.cat([torch.arange(m - rows, m, device="cuda") for m in (77, 300)])
    x, plain, out = torch.randn((n, DIM), device="cuda"), torch.empty((n, DIM), device="cuda"), torch.empty((n, DIM), device="cuda")
    calls = layer.calls(step)
    before = cache.data.clone()
    layer.forward(x, calls, plain)
    torch.cuda.synchronize()
    # the projections' rows as the plain step left them
    q, k, v = (calls.buffers[w].clone() for w in "qkv")
    cache.data.copy_(before)
    seen = []

    def between(q, k, v, stream):
        seen.append((tuple(q.shape), tuple(k.shape), tuple(v.shape), stream))
        _rotate(q, pos), _rotate(k, pos)
    layer.forward(x, calls, out, between=between)
    torch.cuda.synchronize()
    assert seen == [((n, HEADS, HD), (n, KV, HD), (n, KV, HD), None)]
    _rotate(q, pos), _rotate(k, pos)
    got = cache.data.clone()
    cache.data.copy_(before)
    o = torch.empty((n, HEADS, HD), device="cuda")
    attn.Append(cache, 0, step, k, v).run()
    (attn.TokenAttention if rows == 1 else attn.ChunkAttention)(cache, 0, step, q, o).run()
    torch.cuda.synchronize()
    assert torch.equal(got, cache.data) and not torch.equal(got, before)
    assert torch.equal(calls.buffers["o"], o)
    assert torch.isfinite(out).all() and not torch.equal(out, plain)
