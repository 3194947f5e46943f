"""osmos_sample's workspace: what it holds before a call does not matter, and calls of other rows, lengths, types and limits take
turns with one workspace, queued on one stream without a wait or captured into graphs. Each call's outputs are compared with those of the
same call on a workspace of its own."""
import ctypes
import math

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

from libosmos_amd import capi, rows  # noqa: E402

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


def _calls():
    """calls whose workspaces lie differently: rows of many slices and of two, counted by value, of one slice (probabilities alone);
    greedy rows, rows of nothing, of one token, of equal logits (more of them than are listed), and every limit among them"""
    out = []
    for i, (n, vocab, kind, probs) in enumerate([(7, 200003, F32, True), (300, 33001, BF16, False), (5, 40009, F16, True), (1, 1 << 20, F32, False),
                                                 (9, 33000, F32, True), (40, 5000, BF16, True), (64, 70001, F32, False), (2, 300000, F16, False)]):
        g = torch.Generator(device="cuda")
        g.manual_seed(100 + i)
        x = (2.5 * torch.randn((n, vocab), generator=g, device="cuda")).to(kind)
        f = lambda: torch.rand(n, generator=g, device="cuda")  # noqa: E731
        args = dict(temperature=torch.where(f() < 0.3, 0.0, 0.5 + f()), top_k=torch.where(f() < 0.5, 0.0, 1 + f() ** 4 * vocab).int(),
                    top_p=torch.where(f() < 0.4, 1.0, 0.2 + 0.79 * f()), min_p=torch.where(f() < 0.4, 0.0, 10.0 ** (-16 * f())))
        if n > 4:
            x[0] = -math.inf
            x[1] = math.nan
            x[2] = -1.5
            x[3, :-1] = -math.inf
            x[4, : vocab // 2] = torch.finfo(kind).min
        u = f()
        buffers = []
        for _ in "ab":  # the call's own outputs, and those to compare with
            e = lambda t, *s: torch.full(s, -5, dtype=t, device="cuda")  # noqa: E731
            buffers.append((e(torch.int32, n), dict(prob=e(F32, n), kept=e(torch.int32, n), **(dict(probs=e(F32, n, vocab)) if probs else {}))))
        alone = rows.Sample(x, u, buffers[1][0], **args, **buffers[1][1])
        alone.run()
        out.append((rows.Sample(x, u, buffers[0][0], **args, **buffers[0][1]), buffers))
    torch.cuda.synchronize()
    return out


def _same(buffers, what):
    (token, own), (token2, want) = buffers
    assert torch.equal(token, token2), what
    for name in own:
        assert torch.equal(own[name].view(torch.int32), want[name].view(torch.int32)), (what, name)


def _queue(call, ws, stream=None):
    assert capi.lib().osmos_sample(ctypes.byref(call.desc), capi.addr(ws), ws.numel(), stream)


@pytest.mark.parametrize("fill", [0x00, 0x01, 0x7F, 0xFF])
def test_what_it_held(fill):
    print(hex(fill), flush=True)
    for i, (call, buffers) in enumerate(_calls()):
        need = capi.lib().osmos_sample_workspace(ctypes.byref(call.desc))
        ws = torch.full((need + 256,), fill, dtype=torch.uint8, device="cuda")
        buffers[0][0].fill_(-9)
        torch.cuda.synchronize()
        assert capi.lib().osmos_sample(ctypes.byref(call.desc), capi.addr(ws), need, None)
        torch.cuda.synchronize()
        _same(buffers, (fill, i))
        assert (ws[need:] == fill).all()


def test_shared_by_calls_in_turn():
    calls = _calls()
    need = max(capi.lib().osmos_sample_workspace(ctypes.byref(c.desc)) for c, _ in calls)
    ws = torch.full((need,), 0xFF, dtype=torch.uint8, device="cuda")
    order = [0, 1, 2, 3, 4, 5, 6, 7, 7, 6, 5, 4, 3, 2, 1, 0, 3, 6, 1, 4, 7, 2, 5, 0]
    for i in order[:8], order[8:16], order[16:]:
        for call, buffers in calls:
            buffers[0][0].fill_(-9)
        torch.cuda.synchronize()
        for j in i:
            _queue(calls[j][0], ws)
        torch.cuda.synchronize()
        for j, (call, buffers) in enumerate(calls):
            _same(buffers, (i, j))


def test_shared_by_graphs():
    """two graphs of different calls over one workspace, replayed in turn on one stream"""
    calls = _calls()[:4]
    need = max(capi.lib().osmos_sample_workspace(ctypes.byref(c.desc)) for c, _ in calls)
    ws, s, graphs = torch.full((need,), 0xFF, dtype=torch.uint8, device="cuda"), torch.cuda.Stream(), []
    for pair in (calls[:2], calls[2:]):
        g = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(g, stream=s):
            for call, _ in pair:
                _queue(call, ws, s.cuda_stream)
        graphs.append(g)
    for i in range(4):
        for call, buffers in calls:
            buffers[0][0].fill_(-9)
        torch.cuda.synchronize()
        with torch.cuda.stream(s):
            for g in graphs if i % 2 else graphs[::-1]:
                g.replay()
        torch.cuda.synchronize()
        for j, (call, buffers) in enumerate(calls):
            _same(buffers, (i, j))
