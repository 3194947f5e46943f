"""osmos_norm against its formula: every output bit for bit, the row's sum of squares in float64 (include/osmos_rows.h); the tiles
and the codes against mm_x16 and q8_round of the float rows."""
import ctypes
import math

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

from libosmos_amd import capi, rows  # noqa: E402

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


def _bits(t):
    return t.contiguous().view({4: torch.int32, 2: torch.int16, 1: torch.int8}[t.element_size()])


def _same(got, want, what):
    """the same bits (any NaN for a NaN)"""
    assert got.dtype == want.dtype and got.shape == want.shape, what
    ok = (_bits(got) == _bits(want)) | (torch.isnan(got) & torch.isnan(want) if got.is_floating_point() else False)
    assert ok.all(), "%s: %d of %d differ" % (what, int((~ok).sum()), ok.numel())


def _formula(x, add, weight, eps, offset):
    s = x.float() if add is None else x.float() + add.float()
    d = s.double()
    r = (1.0 / torch.sqrt((d * d).sum(1, keepdim=True) / s.shape[1] + eps)).float()
    w = torch.ones(s.shape[1], device="cuda") if weight is None else weight.float()
    return s, s * r * (w + torch.tensor(offset, device="cuda"))


def _make(n, dim, kind, seed=0, pad=0, rms=1.0):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return (torch.randn((n, dim + pad), generator=g, device="cuda") * rms).to(kind)[:, :dim]


@pytest.mark.parametrize("n,dim", [(1, 1), (1, 7), (3, 64), (5, 255), (2, 256), (17, 1000), (1, 2048), (33, 4096), (2, 4097), (3, 6144), (9, 8192),
                                   (1, 16384), (2, 40001), (1, 65536), (700, 96), (300, 1536)])
@pytest.mark.parametrize("kind", [F32, F16, BF16], ids=str)
def test_rows(n, dim, kind):
    print(n, dim, kind, flush=True)
    pad = 5 if dim % 2 else 0
    x, add, w = _make(n, dim, kind, 1, pad, 3.0), _make(n, dim, kind, 2, pad), _make(1, dim, kind, 3)[0].contiguous()
    for out_kind in (F32, F16, BF16):
        total = torch.full((n, dim + pad), 7.0, dtype=kind, device="cuda")
        out = torch.full((n, dim + 3), 7.0, dtype=out_kind, device="cuda")
        rows.Norm(x, add=add, sum=total[:, :dim], weight=w, out=out[:, :dim], eps=1e-5, offset=0.5).run()
        s, y = _formula(x, add, w, 1e-5, 0.5)
        _same(total[:, :dim], s.to(kind), "sum")
        _same(out[:, :dim], y.to(out_kind), "out")
        assert (out[:, dim:] == 7).all() and (total[:, dim:] == 7).all()  # (what lies between the rows is left)
    rows.Norm(x, out=out[:, :dim], eps=0.0).run()
    _same(out[:, :dim], _formula(x, None, None, 0.0, 0.0)[1].to(out_kind), "no weight")


@pytest.mark.parametrize("n,dim", [(1, 32), (15, 2048), (16, 512), (17, 4096), (40, 5120), (1, 8192), (130, 96)])
@pytest.mark.parametrize("kind", [F32, F16, BF16], ids=str)
def test_tiles_and_codes(n, dim, kind):
    print(n, dim, kind, flush=True)
    x, add, w = _make(n, dim, kind, 4, 3, 2.0), _make(n, dim, kind, 5), _make(1, dim, F32, 6)[0].contiguous()
    tiles = (n + 15) // 16 * 16 * dim
    x16, over = torch.full((tiles,), 9.0, dtype=F16, device="cuda"), torch.zeros(1, dtype=torch.int32, device="cuda")
    codes, scales = torch.full((n, dim), 99, dtype=torch.int8, device="cuda"), torch.full((n, dim // 32), 9.0, device="cuda")
    out, total = torch.empty((n, dim), device="cuda"), add  # (in place: the sum over what was added)
    want_sum, y = _formula(x, add, w, 1e-6, 0.0)
    rows.Norm(x, add=add, sum=total, weight=w, out=out, x16=x16, overflow=over, codes=codes, scales=scales).run()
    _same(out, y, "out")
    _same(total, want_sum.to(kind), "sum in place")
    want16, over2 = torch.full_like(x16, 5.0), torch.zeros_like(over)
    want_codes, want_scales = torch.empty_like(codes), torch.empty_like(scales)
    L, a = capi.lib(), capi.addr
    assert L.mm_x16(a(out), dim, n, dim, a(want16), a(over2), None) and L.q8_round(a(out), n, dim, dim, a(want_codes), a(want_scales), None)
    _same(x16, want16, "tiles")
    _same(codes, want_codes, "codes")
    _same(scales, want_scales, "scales")
    assert int(over) == int(over2) == 0


def test_only_the_sum():
    x, add = _make(3, 77, F32, 1), _make(3, 77, F32, 2)
    total = torch.empty_like(x)
    rows.Norm(x, add=add, sum=total).run()
    _same(total, x + add, "sum")


def test_sum_into_x():
    x, add = _make(5, 512, BF16, 1, 8), _make(5, 512, BF16, 2)
    s, y = _formula(x, add, None, 1e-6, 0.0)
    out = torch.empty((5, 512), device="cuda")
    rows.Norm(x, add=add, sum=x, out=out).run()
    _same(x.contiguous(), s.to(BF16), "sum in place")
    _same(out, y, "out of the sum before its rounding")


@pytest.mark.parametrize("dim", [64, 4096])
def test_overflow(dim):
    """a value past float16's range sets the flag and becomes an infinity, as in mm_x16; nothing clears it"""
    x = _make(3, dim, F32, 1)
    w = torch.ones(dim, device="cuda")
    x16, over = torch.empty(16 * dim, dtype=F16, device="cuda"), torch.zeros(1, dtype=torch.int32, device="cuda")
    call = rows.Norm(x, weight=w, x16=x16, overflow=over)
    call.run()
    assert int(over) == 0
    w[5] = 1e6
    call.run()
    assert int(over) == 1 and torch.isinf(x16).any()
    w[5] = 1.0
    call.run()
    assert int(over) == 1


def test_extremes():
    """squares past float's range, tiny rows, a row of zeros, infinities and NaN in rows that do not touch the others"""
    dim = 256
    x = _make(7, dim, F32, 1)
    x[1] *= 1e30
    x[2] *= 1e-30
    x[3] = 0.0
    x[4, 3] = math.inf
    x[5, 9] = math.nan
    out = torch.empty_like(x)
    rows.Norm(x, out=out, eps=0.0).run()
    y = _formula(x, None, None, 0.0, 0.0)[1]
    _same(out, y, "extremes")
    assert torch.isfinite(out[[0, 1, 2, 6]]).all() and torch.isnan(out[3]).all() and (out[4, :3] == 0).all() and torch.isnan(out[4, 3])
    rows.Norm(x, out=out).run()
    assert (out[3] == 0).all()


def test_a_row_alone():
    """the bits of a row do not depend on how many there are"""
    x, w = _make(3000, 1536, BF16, 1), _make(1, 1536, F32, 2)[0].contiguous()
    out, one = torch.empty((3000, 1536), device="cuda"), torch.empty((1, 1536), device="cuda")
    rows.Norm(x, weight=w, out=out).run()
    for i in (0, 1499, 2999):
        rows.Norm(x[i:i + 1], weight=w, out=one).run()
        _same(one, out[i:i + 1], "row %d" % i)


def test_captured():
    x, add, w = _make(20, 2048, F32, 1), _make(20, 2048, F32, 2), _make(1, 2048, F32, 3)[0].contiguous()
    total, out = torch.empty_like(x), torch.empty((20, 2048), dtype=F16, device="cuda")
    call = rows.Norm(x, add=add, sum=total, weight=w, out=out)
    call.run()
    torch.cuda.synchronize()
    g, s = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.graph(g, stream=s):
        call.run(s.cuda_stream)
    for i in range(4):
        x.copy_(_make(20, 2048, F32, 10 + i))
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        t, y = _formula(x, add, w, 1e-6, 0.0)
        _same(out, y.to(F16), "replay %d" % i)
        _same(total, t, "replay %d" % i)


def test_refusals():
    x = _make(4, 64, F32)
    out = torch.empty_like(x)
    for bad, kind in ((dict(out=out[:3]), ValueError), (dict(out=out.double()), TypeError), (dict(add=x.half(), out=out), TypeError),
                      (dict(weight=x[0][::2], out=out), TypeError), (dict(out=out.t()), TypeError), (dict(codes=out.char()), ValueError),
                      (dict(x16=torch.empty(4 * 64, dtype=F16, device="cuda"), overflow=torch.zeros(1, dtype=torch.int32, device="cuda")), TypeError),
                      (dict(x16=torch.empty(16 * 64, dtype=F16, device="cuda")), ValueError), (dict(out=out.cpu()), TypeError)):
        with pytest.raises(kind):
            rows.Norm(x, **bad)
    for bad in (dict(), dict(out=out, eps=-1.0)):
        with pytest.raises(RuntimeError):
            rows.Norm(x, **bad).run()
    d = rows.Norm(x, out=out).desc
    d.dim = 0
    assert not capi.lib().osmos_norm(ctypes.byref(d), None)
