"""osmos_sample against its definition in float64: tokens and counts equal, probabilities to float's rounding (half a step each for the
weight and for what it is multiplied by). Seeded rows whose choice hangs on less than 1e-9 of the sum would say nothing: there
are none, which is asserted."""
import math

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
import numpy as np  # noqa: E402

from libosmos_amd import rows  # noqa: E402

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


def _one(l, t, k, p, m, u):
    """(token, prob, kept, probs, margin) of a row of logits"""
    l = l.astype(np.float64)
    l = np.where(np.isnan(l), -np.inf, np.minimum(l, 3.4028234663852886e38))
    probs = np.zeros(len(l))
    order = np.argsort(-l, kind="stable")
    order = order[l[order] > -np.inf]
    if len(order) == 0:
        return -1, 0.0, 0, probs, 1.0
    if not t > 0:
        probs[order[0]] = 1
        return int(order[0]), 1.0, 1, probs, 1.0
    w = np.exp((l[order] - l[order[0]]) / t) if not math.isinf(t) else np.ones(len(order))
    margin = 1.0
    n = len(order) if k <= 0 else min(k, len(order))
    if p < 1:
        c = np.cumsum(w[:n])
        goal = max(p, 0.0) * c[-1]
        before = c - w[:n]
        margin = min(margin, np.abs(before[1:] - goal).min() / c[-1] if n > 1 else 1.0)
        n = max(1, int((before < goal).sum()))
    if m > 0:
        margin = min(margin, np.abs(w[:n] / min(m, 1.0) - 1.0)[w[:n] != 1.0].min(initial=1.0))
        n = max(1, min(n, int((w >= min(m, 1.0)).sum())))
    c = np.cumsum(w[:n])
    u = 0.0 if not u > 0 else min(u, 0.99999994)
    at = min(int((c <= u * c[-1]).sum()), n - 1)
    if u > 0:
        margin = min(margin, np.abs(c[:-1] - u * c[-1]).min(initial=math.inf) / c[-1])
    probs[order[:n]] = w[:n] / c[-1]
    return int(order[at]), w[at] / c[-1], n, probs, margin


def _check(logits, u, temperature=None, top_k=None, top_p=None, min_p=None, what="", only=None, exact=False):
    n, dev = logits.shape[0], "cuda"
    f = lambda v, t: None if v is None else torch.tensor(v, dtype=t, device=dev) if isinstance(v, list) else v  # noqa: E731
    u, temperature, top_p, min_p, top_k = f(u, F32), f(temperature, F32), f(top_p, F32), f(min_p, F32), f(top_k, torch.int32)
    token, kept = (torch.full((n,), -7, dtype=torch.int32, device=dev) for _ in "ab")
    prob, probs = torch.full((n,), 7.0, device=dev), torch.full(logits.shape, 7.0, device=dev)
    args = dict(temperature=temperature, top_k=top_k, top_p=top_p, min_p=min_p)
    rows.Sample(logits, u, token, prob=prob, kept=kept, probs=probs, **args).run()
    again = torch.empty_like(token)
    rows.Sample(logits, u, again, **args).run()
    torch.cuda.synchronize()
    assert torch.equal(token, again), what
    host = lambda x, d: np.full(n, d) if x is None else x.double().cpu().numpy()  # noqa: E731
    par = zip(host(temperature, 1.0), host(top_k, 0), host(top_p, 1.0), host(min_p, 0.0), host(u, 0.0))
    at = range(n) if only is None else only
    l = dict(zip(at, logits[torch.tensor(list(at), device=dev)].float().cpu().numpy()))
    for i, (t, k, p, m, v) in enumerate(par):
        if i not in l:
            continue
        tok, pr, ke, want, margin = _one(l[i], t, int(k), p, m, v)
        note = "%s row %d: T %g k %d p %g min %g u %g" % (what, i, t, k, p, m, v)
        assert exact or margin > 1e-9, note
        assert int(token[i]) == tok and int(kept[i]) == ke, "%s: token %d kept %d, wanted %d %d" % (note, token[i], kept[i], tok, ke)
        assert abs(float(prob[i]) - pr) <= 2.0 ** -23 * pr, note
        got = probs[i].double().cpu().numpy()
        # (weights under 2^-44 of the greatest count as zero)
        assert (np.abs(got - want) <= 2.0 ** -23 * want + (want < 2.0 ** -43 * want.max()) * want).all(), note
        assert ((got > 0) <= (want > 0)).all(), note
    return token


def _logits(n, vocab, kind, seed, std=2.5):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    x = std * torch.randn((n, vocab), generator=g, device="cuda")
    x[:, ::97] += 6.0 * torch.rand((n, len(range(0, vocab, 97))), generator=g, device="cuda")
    return x.to(kind), torch.rand(n, generator=g, device="cuda")


def _params(n, vocab, seed):
    r = np.random.default_rng(seed)
    pick = lambda *o: [float(o[i]) for i in r.integers(0, len(o), n)]  # noqa: E731
    return dict(temperature=[0.0 if r.random() < 0.1 else float(r.uniform(0.2, 2.0)) for _ in range(n)],
                top_k=[int(x) for x in np.where(r.random(n) < 0.5, 0, 1 + (r.random(n) ** 3 * vocab).astype(int))],
                top_p=[1.0 if r.random() < 0.4 else float(r.uniform(0.05, 0.999)) for _ in range(n)], min_p=pick(0, 0, 0, 0.01, 0.1, 0.5))


@pytest.mark.parametrize("n,vocab", [(40, 1), (40, 2), (30, 63), (30, 1000), (20, 4097), (12, 32003), (9, 100352), (5, 151001), (4, 262144), (40, 65536),
                                     (150, 20000)])
@pytest.mark.parametrize("kind", [F32, F16, BF16], ids=str)
def test_mixed(n, vocab, kind):
    print(n, vocab, kind, flush=True)
    x, u = _logits(n, vocab, kind, vocab + n)
    _check(x, u, what="mixed", **_params(n, vocab, vocab))


@pytest.mark.parametrize("n,vocab", [(270, 40009), (600, 65544), (180, 98311)])
def test_many_rows_by_value(n, vocab):
    """bf16 rows in such numbers that their tokens are counted by value, in slices of one round and of more; values outside the
    counted range (256 and more, under 2^-24, zeros, infinities, NaN) among them, and rows of nothing else"""
    print(n, vocab, flush=True)
    x, u = _logits(n, vocab, BF16, n)
    p = _params(n, vocab, n)
    only = [0, 1, 2, 3, 4, 5, 6, 7, 8, 9, n // 2, n - 1]
    for i in (1, n - 1):
        x[i, ::3] = -math.inf
    x[2, 5::7] = 1e-9
    x[2, 6::7] = 0.0
    x[3, 1000], x[3, vocab - 1], x[3, 2000:2100] = 300.0, 300.0, 299.0
    x[4] = -500.0
    x[4, 777::5] = -499.0
    x[5] = -0.0
    x[6] = math.nan
    x[6, vocab - 3] = 3.0
    x[7] = -math.inf
    x[8, 11], x[8, 12] = math.inf, math.nan
    x[9, 40::2] = torch.finfo(BF16).min
    for i in (2, 3, 4, 5):
        p["temperature"][i] = 1.0
    p["temperature"][n // 2] = 0.0
    _check(x, u, what="by value", only=only, exact=True, **p)
    _check(x, u, what="by value, no limits", only=only, exact=True)


def test_largest_vocab():
    x, u = _logits(2, 1 << 20, F32, 3)
    _check(x, u, top_p=[0.9, 1.0], top_k=[0, 300000], what="2^20")


@pytest.mark.parametrize("kind", [F32, BF16], ids=str)
def test_one_limit_each(kind):
    x, u = _logits(8, 50257, kind, 5)
    _check(x, u, what="none")
    _check(x, u, top_k=[1, 2, 5, 40, 1000, 50256, 50257, 60000], what="k")
    _check(x, u, top_p=[1e-6, 0.1, 0.5, 0.9, 0.99, 0.9999, 1.0, 2.0], what="p")
    _check(x, u, min_p=[1.0, 0.5, 0.1, 0.01, 1e-4, 1e-8, 1.5, -1.0], what="min-p")
    _check(x, u, temperature=[0.01, 0.1, 0.5, 1.0, 2.0, 10.0, 1000.0, 1e20], what="T")


def test_strides_and_no_outputs():
    x, u = _logits(6, 5000, BF16, 8)
    wide = torch.full((6, 5011), 30.0, dtype=BF16, device="cuda")
    wide[:, 3:5003] = x
    t = _check(wide[:, 3:5003], u, top_k=[50] * 6)
    assert torch.equal(t, _check(x, u, top_k=[50] * 6))


def test_equal_logits():
    """ties: the lower index first, the kept ones a prefix of the indexes"""
    n = 6
    for vocab in (1, 7, 5000, 140000):
        x = torch.full((n, vocab), -3.25, device="cuda")
        u = [0.0, 0.1, 0.37, 0.5, 0.77, 0.99]
        got = _check(x, u, what="all alike", exact=True)
        assert got.tolist() == [min(vocab - 1, math.floor(float(np.float32(v)) * vocab)) for v in u]
        got = _check(x, u, top_k=[3] * n, what="k of all alike", exact=True)
        assert got.tolist() == [min(min(3, vocab) - 1, math.floor(float(np.float32(v)) * min(3, vocab))) for v in u]
    x = torch.full((2, 9000), 1.0, device="cuda")
    x[:, 100::3] = 2.0  # 2967 of them
    x[:, 5000] = 5.0
    _check(x, [0.4, 0.9], top_k=[1500, 4000], temperature=[2.0, 3.0], what="ties at the border")
    _check(x, [0.4, 0.9], top_p=[0.3, 0.8], temperature=[2.0, 3.0], what="ties at the border")


@pytest.mark.parametrize("kind", [F32, F16, BF16], ids=str)
def test_masked(kind):
    inf, low = math.inf, torch.finfo(kind).min
    x, u = _logits(9, 3001, kind, 11)
    x[0] = -inf                       # nothing left
    x[1] = math.nan
    x[2, :] = -inf
    x[2, 2999] = -5.0                 # one left
    x[3, 1::2] = -inf
    x[4, 1::2] = math.nan
    x[5, 7:] = low
    x[6] = low                        # all at the lowest value: alike
    x[7, 17] = inf
    x[7, 2000] = inf                  # two that take it all
    x[8, :] = -inf
    x[8, 5], x[8, 6] = low, 0.0
    for args in (dict(), dict(top_k=[4] * 9), dict(top_p=[0.7] * 9), dict(min_p=[0.05] * 9), dict(temperature=[0.0] * 9), dict(temperature=[0.5] * 9, top_k=[100] * 9, top_p=[0.9] * 9, min_p=[0.01] * 9)):
        got = _check(x, u, what="masked %s" % args, exact=True, **args)
        assert got[:3].tolist() == [-1, -1, 2999] and int(got[8]) in (6,)


def test_odd_parameters():
    nan, inf = math.nan, math.inf
    x, u = _logits(10, 4000, F32, 13)
    _check(x, u, temperature=[nan, -1.0, 0.0, -0.0, inf, 1e-30, 1e-38, 1e-45, 3e38, 1e-3], what="T")
    _check(x, u, top_p=[nan, -1.0, 0.0, 1.0, inf, -inf, 1e-30, 0.5, 0.25, 0.125], what="p")
    _check(x, u, min_p=[nan, -1.0, 0.0, 1.0, inf, -inf, 1e-30, 0.5, 2.0, 0.125], what="min-p")
    _check(x, u, top_k=[0, -1, -2 ** 31, 2 ** 31 - 1, 1, 3999, 4000, 4001, 2, 3], what="k")
    _check(x, [0.0, -1.0, nan, 1.0, 5.0, inf, -inf, 0.99999994, 1e-30, 0.5], top_k=[10] * 10, what="u", exact=True)


@pytest.mark.parametrize("scale", [1e-6, 1e-2, 100.0, 1e5, 1e30])
def test_magnitudes(scale):
    """logits far from the usual size, and temperatures that bring them back or do not"""
    x, u = _logits(6, 20001, F32, 17)
    x = x * scale
    _check(x, u, temperature=[1.0, scale, scale * 0.3, scale * 2, 0.7, 1.0 / scale if scale < 1e20 else 1.0], top_p=[0.95] * 6, what="size %g" % scale,
           exact=True)
    _check(x - 1000.0 * min(scale, 1e6), u, temperature=[scale] * 6, top_k=[77] * 6, what="size %g, far from zero" % scale, exact=True)


@pytest.mark.parametrize("vocab", [4000, 40000])
def test_weights_of_almost_nothing(vocab):
    """limits that end among tokens of 2^-43 of the greatest weight and less, which add little or nothing to the sums"""
    x = torch.full((6, vocab), -60.0, device="cuda")
    x[:, 7] = 0.0
    x[:, 100:3100] = -29.4 - 1.1e-3 * torch.arange(3000, device="cuda")
    u = [0.3, 0.9, 0.99999, 0.5, 0.99999994, 0.0]
    got = _check(x, u, top_k=[1500, 2900, 3001, 1025, 40, vocab - 1], what="k", exact=True)
    assert got.tolist() == [7] * 6
    x[3:, 8] = -0.5
    _check(x, u, top_k=[1500, 2900, 3001, 1025, 2000, 2500], top_p=[0.5, 0.99, 0.999999, 0.9, 0.7, 0.3], what="k, p", exact=True)
    _check(x, u, top_k=[1500, 0, 3001, 1025, 2000, 2500], min_p=[1e-13, 2e-13, 5e-14, 1e-13, 1.0, 0.6], what="k, min-p", exact=True)


def test_denormal_logits():
    """logits and temperatures among float's least values"""
    for scale in (1e-38, 1e-41, 1e-43):
        for vocab in (3000, 50001):
            x, u = _logits(4, vocab, F32, 37)
            x = (x.double() * scale).float()
            t = [float(np.float32(scale))] * 4
            _check(x, u, temperature=t, what="size %g" % scale, exact=True)
            _check(x, u, temperature=t, top_p=[0.9] * 4, min_p=[0.0, 0.01, 0.1, 0.5], what="size %g" % scale, exact=True)
            _check(x, u, temperature=t, top_k=[40, 2000, 5, 1], what="size %g" % scale, exact=True)


def test_a_row_alone():
    x, u = _logits(64, 70001, F32, 19)
    p = _params(64, 70001, 23)
    all_rows = _check(x, u, what="together", **p)
    for i in (0, 31, 63):
        got = _check(x[i:i + 1], u[i:i + 1], what="alone", **{k: v[i:i + 1] for k, v in p.items()})
        assert int(got) == int(all_rows[i])


def test_frequencies():
    """evenly spread numbers draw every token as often as its probability says, to one draw"""
    n, vocab = 5000, 12
    x, _ = _logits(1, vocab, F32, 29, 1.0)
    u = (torch.arange(n, device="cuda", dtype=torch.float64) + 0.5).div(n).float()
    token = torch.empty(n, dtype=torch.int32, device="cuda")
    rows.Sample(x.expand(n, vocab).contiguous(), u, token).run()
    want = torch.softmax(x[0].double(), 0) * n
    assert ((torch.bincount(token, minlength=vocab) - want).abs() <= 1.0 + 1e-3).all()


def test_captured_and_side_stream():
    """replays with other logits between them, the workspace shared with an eager call on the same stream"""
    x, u = _logits(3, 150001, F32, 31)
    token, want = torch.empty(3, dtype=torch.int32, device="cuda"), torch.empty(3, dtype=torch.int32, device="cuda")
    k = torch.tensor([0, 50, 1000], dtype=torch.int32, device="cuda")
    p = torch.tensor([0.9, 1.0, 0.8], device="cuda")
    call, plain = rows.Sample(x, u, token, top_k=k, top_p=p), rows.Sample(x, u, want, top_k=k, top_p=p)
    s = torch.cuda.Stream()
    torch.cuda.synchronize()
    call.run(s.cuda_stream)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        call.run(s.cuda_stream)
    for i in range(5):
        y, v = _logits(3, 150001, F32, 40 + i)
        x.copy_(y)
        u.copy_(v)
        token.fill_(-9)
        plain.run()
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(token, want), i
        assert len(set(token.tolist())) == 3


def test_refusals():
    x, u = _logits(4, 100, F32, 1)
    token = torch.empty(4, dtype=torch.int32, device="cuda")
    for args, kw, kind in (((x, u[:3], token), {}, TypeError), ((x, u.double(), token), {}, TypeError), ((x, u, token.long()), {}, TypeError),
                           ((x.t(), u, token), {}, TypeError), ((x.double(), u, token), {}, TypeError), ((x, u, token), dict(top_k=u), TypeError),
                           ((x, u, token), dict(probs=x[:, :50]), ValueError), ((x, u, token), dict(probs=x.half()), TypeError),
                           ((x, u, token.cpu()), {}, TypeError), ((x[None], u, token), {}, TypeError)):
        with pytest.raises(kind):
            rows.Sample(*args, **kw)
    with pytest.raises(RuntimeError):
        rows.Sample(torch.zeros((1, (1 << 20) + 1), device="cuda"), u[:1], token[:1]).run()
