"""A plain float64 statement of the attention and of the paged cache for the tests (torch, any device), and the error that
the kernels' arithmetic may make (products of 16-bit values, sums and softmax in float32)."""
import math

import torch

UNIT = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}


def rows_of_pages(data, scale, layer, which, table, n, head):
    """tokens 0 .. n - 1 of a sequence's keys (0) or values (1) in float64, and which of them are in a page that exists"""
    pages, page = data.shape[2], data.shape[4]
    at = torch.arange(n, device=data.device)
    ids = table[at // page].long()
    here = (ids >= 0) & (ids < pages)
    plane = data[layer, which].view(torch.uint8) if data.dtype == torch.float8_e4m3fn else data[layer, which]
    x = plane[ids.clamp(0, pages - 1), head, at % page]
    x = (x.view(data.dtype) if data.dtype == torch.float8_e4m3fn else x).double()
    if scale is not None:
        x = x * scale[layer, which, head].double()
    return x, here


def attend(q, k, v, pos, here, scale, window, dtype, out_dtype):
    """one head: q (r, d) at positions pos over k, v (n, d), all float64. (out, lse, the error allowed in out, in lse)"""
    n = k.shape[0]
    key = torch.arange(n, device=q.device)
    seen = (key <= pos[:, None]) & here
    if window:
        seen &= key > pos[:, None] - window
    kz, vz = torch.where(here[:, None], k, 0.0), torch.where(here[:, None], v, 0.0)
    x = (q @ kz.T) * scale
    size = (q.abs() @ kz.abs().T) * scale  # the sums of the products' magnitudes
    x = torch.where(seen, x, -math.inf)
    top = x.amax(1, keepdim=True) if n else x.new_zeros((q.shape[0], 1))
    top = torch.where(torch.isfinite(top), top, 0.0)
    p = torch.exp(x - top)
    total = p.sum(1, keepdim=True)
    p = p / total.clamp(min=1e-300)
    live = seen.any(1)
    out = torch.where(live[:, None], p @ vz, 0.0)
    lse = torch.where(live, top[:, 0] + torch.log(total[:, 0].clamp(min=1e-300)), -math.inf)
    # a score's error: the sum of dim products in float32 (a rounding each), its scaling to base 2 and the subtraction
    size = torch.where(seen, size, 0.0).amax(1) if n else x.new_zeros(q.shape[0])
    ds = (q.shape[1] + 8) * 2.0 ** -24 * size + size * 2.0 ** -22 + 2.0 ** -21
    weight = p @ vz.abs()
    most = vz.abs().amax() if n else 0.0
    # the probabilities' rounding (against the running maximum: below 2^-14 an absolute 2^-25 in f16), the scores' errors in
    # p and in the sum, the running sums
    e = (UNIT[dtype] + 2 * ds[:, None] + (n + 64) * 2.0 ** -24) * weight + n * 2.0 ** -25 * most
    e = e + (out.abs() + e) * UNIT[out_dtype] + 2.0 ** -24  # the output's rounding (f16's least step)
    el = ds + (n + 64) * 2.0 ** -24 + lse.abs().nan_to_num(0.0, 0.0, 0.0) * 2.0 ** -22
    return out, lse, e, el


def check(got, lse, want, wlse, tol, ltol, what):
    got, lse = got.double(), lse.double()
    bad = ~((got - want).abs() <= tol)
    assert not bad.any(), "%s: %d of %d values off, worst %.3g where %.3g is allowed" % (
        what, int(bad.sum()), bad.numel(), float((got - want).abs()[bad].nan_to_num(9e9).max()), float(tol[bad].max()))
    dead = torch.isneginf(wlse)
    assert torch.equal(torch.isneginf(lse), dead), what
    off = (lse - wlse).abs()[~dead]
    assert (off <= ltol[~dead]).all(), "%s: lse off by %.3g" % (what, float(off.max()))
