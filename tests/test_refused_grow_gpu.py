"""A step queued behind an osmos_kv_grow that the pool could not carry out, its `done` as the step's `live`: no page is written for
a refused sequence (whose last tokens lie in pages that others hold too), its rows attend to nothing, and the granted ones are as
they would be alone."""
import ctypes

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
from tests import attn_ref  # noqa: E402

HEADS, KV, DIM, PAGE = 4, 2, 64, 16


def _ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _granted(data, pool, s, q, out, lse, what):
    """the rows q of sequence s, its last, against a float64 statement"""
    m, r = int(pool.len[s]), q.shape[0]
    pos = torch.arange(m - r, m, device="cuda")
    for h in range(HEADS):
        (k, here), (v, _) = (attn_ref.rows_of_pages(data, None, 0, w, pool.table[s], m, h // (HEADS // KV)) for w in (0, 1))
        want = attn_ref.attend(q[:, h].double(), k, v, pos, here, DIM ** -0.5, 0, torch.float16, torch.float16)
        attn_ref.check(out[:, h], lse[:, h], *want, (what, s, h))


@pytest.mark.parametrize("rows", [1, 20])
def test_forked_sequences_in_a_full_pool(rows):
    """a prompt, three children that share its pages, free pages for some of them only: nothing of what is there changes"""
    from libosmos_amd import attn
    g = _gen(rows)
    # 33 tokens a sequence in 3 pages, the last shared: 1 row more needs a copy of it; 20 more a copy and another page, but for the
    # last of the holders
    for free in range(5 if rows == 1 else 8):
        pages = 3 + free
        data = torch.randn((1, 2, pages, KV, PAGE, DIM), generator=g, device="cuda").half()
        cache = attn.KvCache(data)
        pool = attn.KvPool.empty(cache, 4, 8 * PAGE)
        pool.grow(_ints([2]), _ints([33]))
        pool.fork(_ints([2, 2, 2]), _ints([0, 1, 3]))
        torch.cuda.synchronize()
        before, order = data.clone(), [3, 1, 2, 0]
        done = _ints([7] * 4)
        pool.grow(_ints(order), _ints([rows] * 4), done)
        n = 4 * rows
        k, v, q = (torch.randn((n, h, DIM), generator=g, device="cuda").half() for h in (KV, KV, HEADS))
        step = attn.KvStep(_ints([i * rows for i in range(5)]), pool.len, pool.table, n_tok=n, max_tok=rows, max_len=8 * PAGE,
                           seq=_ints(order), live=done)
        out, lse = torch.full_like(q, 7.0), torch.full((n, HEADS), 7.0, device="cuda")
        print("full pool", rows, free, flush=True)
        attn.Append(cache, 0, step, k, v).run()
        (attn.TokenAttention if rows == 1 else attn.ChunkAttention)(cache, 0, step, q, out, lse).run()
        torch.cuda.synchronize()
        granted = done.tolist()
        need = [1, 1, 1, 0] if rows == 1 else [2, 2, 2, 1]
        want, left = [], free
        for x in need:
            left = left - x if x <= left and all(want) else -1
            want.append(int(left >= 0))
        assert granted == want
        # what the granted ones may have changed: their own new tokens' places (a page's copy among them)
        for i, s in enumerate(order):
            at = slice(i * rows, (i + 1) * rows)
            m = int(pool.len[s])
            assert m == 33 + rows * granted[i]
            for p in range(33):  # every old token of every sequence
                page = int(pool.table[s, p // PAGE])
                old = [0, 1, 2][p // PAGE]
                assert torch.equal(data[0, :, page, :, p % PAGE], before[0, :, old, :, p % PAGE]), (s, p)
            if granted[i]:
                page = pool.table[s, torch.arange(33, m, device="cuda") // PAGE].long()
                for w, x in enumerate((k, v)):
                    assert torch.equal(data[0, w][page, :, torch.arange(33, m, device="cuda") % PAGE], x[at])
                _granted(data, pool, s, q[at], out[at], lse[at], free)
            else:
                assert (out[at] == 0).all() and torch.isneginf(lse[at]).all()
        if not any(granted):
            assert torch.equal(data, before)


@pytest.mark.parametrize("token", [True, False])
def test_many_sequences_some_not_live(token):
    """more sequences than a wave has lanes, in another order than the tables', every third not live"""
    from libosmos_amd import attn
    g, n_seq = _gen(5), 130
    rows = [1] * n_seq if token else [1 + i % 5 for i in range(n_seq)]
    data = torch.randn((1, 2, 1000, KV, PAGE, DIM), generator=g, device="cuda").half()
    cache = attn.KvCache(data)
    pool = attn.KvPool.empty(cache, n_seq, 8 * PAGE)
    order = torch.randperm(n_seq, generator=g, device="cuda").int()
    pool.grow(order, _ints([r + (11 * i) % 90 for i, r in enumerate(rows)]))
    live = _ints([int(i % 3 != 1) for i in range(n_seq)])
    n = sum(rows)
    starts = [sum(rows[:i]) for i in range(n_seq + 1)]
    k, v, q = (torch.randn((n, h, DIM), generator=g, device="cuda").half() for h in (KV, KV, HEADS))
    step = attn.KvStep(_ints(starts), pool.len, pool.table, n_tok=n, max_tok=max(rows), max_len=8 * PAGE, seq=order, live=live)
    out, lse, want = torch.full_like(q, 7.0), torch.full((n, HEADS), 7.0, device="cuda"), data.clone()
    lens, table = pool.len.tolist(), pool.table.tolist()
    for i, s in enumerate(order.tolist()):
        for j in range(rows[i] if i % 3 != 1 else 0):
            p, t = lens[s] - rows[i] + j, starts[i] + j
            want[0, 0, table[s][p // PAGE], :, p % PAGE], want[0, 1, table[s][p // PAGE], :, p % PAGE] = k[t], v[t]
    print("not live", token, flush=True)
    attn.Append(cache, 0, step, k, v).run()
    (attn.TokenAttention if token else attn.ChunkAttention)(cache, 0, step, q, out, lse).run()
    torch.cuda.synchronize()
    assert torch.equal(data, want)
    for i, s in enumerate(order.tolist()):
        at = slice(starts[i], starts[i + 1])
        if i % 3 == 1:
            assert (out[at] == 0).all() and torch.isneginf(lse[at]).all()
        else:
            _granted(data, pool, s, q[at], out[at], lse[at], token)


def test_decoding_as_a_graph_until_the_pool_is_full():
    """grow, append and attention captured once and replayed past the last free page: from there on nothing is written"""
    from libosmos_amd import attn
    g = _gen(6)
    data = torch.randn((1, 2, 5, KV, PAGE, DIM), generator=g, device="cuda").half()
    cache = attn.KvCache(data)
    pool = attn.KvPool.empty(cache, 2, 8 * PAGE)
    pool.grow(_ints([0]), _ints([30]))
    pool.fork(_ints([0]), _ints([1]))  # (2 pages of both; the first 9 tokens more take a copy and a third page each: full)
    both, one, done = _ints([0, 1]), _ints([9, 9]), _ints([7, 7])
    k, v, q = (torch.zeros((2, h, DIM), device="cuda").half() for h in (KV, KV, HEADS))
    out, lse = torch.empty_like(q), torch.empty((2, HEADS), device="cuda")
    step = attn.KvStep(_ints([0, 1, 2]), pool.len, pool.table, n_tok=2, max_tok=1, max_len=8 * PAGE, live=done)
    calls = [attn.Append(cache, 0, step, k, v), attn.TokenAttention(cache, 0, step, q, out, lse)]
    torch.cuda.synchronize()
    stream, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    at = ctypes.c_void_p(stream.cuda_stream)
    with torch.cuda.stream(stream):
        graph.capture_begin()
        pool.grow(both, one, done, at)
        for c in calls:
            c.run(at)
        graph.capture_end()
    torch.cuda.synchronize()
    was, outcomes = pool.len.tolist(), []
    for i in range(6):
        for x in (k, v, q):
            x.copy_(torch.randn(x.shape, generator=g, device="cuda"))
        out.fill_(7.0), lse.fill_(7.0)
        before = data.clone()
        print("replay", i, flush=True)
        graph.replay()
        torch.cuda.synchronize()
        granted = done.tolist()
        outcomes.append(granted)
        for s in (0, 1):
            assert int(pool.len[s]) == was[s] + 9 * granted[s]
            if granted[s]:
                m = int(pool.len[s])
                page = int(pool.table[s, (m - 1) // PAGE])
                assert torch.equal(data[0, 0, page, :, (m - 1) % PAGE], k[s])
                assert torch.equal(data[0, 1, page, :, (m - 1) % PAGE], v[s])
                _granted(data, pool, s, q[s:s + 1], out[s:s + 1], lse[s:s + 1], i)
            else:
                assert (out[s] == 0).all() and torch.isneginf(lse[s]).all()
        was = pool.len.tolist()
        if not any(granted):
            assert torch.equal(data, before)
    assert outcomes == [[1, 1]] * 2 + [[0, 0]] * 4
