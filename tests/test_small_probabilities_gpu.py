"""f16 attention where one key takes almost all of the weight and its value is zero, so that the output is what thousands of keys
with probabilities far under f16's least step make together: each row against its closed form."""
import math

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

LOW = -17.5  # every other key's score below the first's: e^-17.5 is 2.5e-8, f16's least step 6.0e-8


def _ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def _check(out, seen):
    """rows that see `seen` keys, the first of score 0 and value 0, the others of score LOW and value 1"""
    many = (seen.double() - 1) * math.exp(LOW)
    want = many / (1 + many)
    # a probability is kept to 11 bits, below 2^-21 of the greatest to 2^-32 of it; sums of n positive values in float32, exp2
    # of a score scaled in float32 (half a unit of 17.5 x log2 e, 2^-20, and the instruction's own), the division
    rel = 2.0 ** -11 + (seen.double() + 64) * 2.0 ** -24 + 2.0 ** -18
    tol = rel * want + seen.double() * 2.0 ** -32
    off = (out.double() - want[:, None, None]).abs()
    assert (off <= tol[:, None, None]).all(), "off by up to %.3g of it" % float((off / want.clamp(min=1e-30)[:, None, None]).max())


@pytest.mark.parametrize("dim", [64, 128, 192, 256])
@pytest.mark.parametrize("cache", ["f16", "f8"])
@pytest.mark.parametrize("rows,n", [(1, 16384), (1, 131072), (3, 16384), (200, 40000)])
def test_pages(rows, n, cache, dim):
    from libosmos_amd import attn
    page, heads = 64, 2
    pages = -(-n // page)
    x = torch.zeros((1, 2, pages, 1, page, dim), device="cuda")
    x[0, 0, :, :, :, 0], x[0, 1] = LOW, 1.0
    x[0, :, 0, 0, 0] = 0.0
    scale = None
    if cache == "f8":  # (17.5 is 1.25 x 14: e4m3 holds 14)
        scale = torch.tensor([[[1.25], [1.0]]], device="cuda")
        x[:, 0] /= 1.25
    c = attn.KvCache(x.to(torch.float16 if cache == "f16" else torch.float8_e4m3fn), scale)
    table = torch.arange(pages, dtype=torch.int32, device="cuda")[None].contiguous()
    q = torch.zeros((rows, heads, dim), dtype=torch.float16, device="cuda")
    q[..., 0] = 1.0
    step = attn.KvStep(_ints([0, rows]), _ints([n]), table, n_tok=rows, max_tok=rows, max_len=n)
    for kind in ((attn.TokenAttention, attn.ChunkAttention) if rows == 1 else (attn.ChunkAttention,)):
        out = torch.empty((rows, heads, dim), device="cuda")
        print("small", kind.__name__, rows, n, cache, dim, flush=True)
        kind(c, 0, step, q, out, scale=1.0).run()
        torch.cuda.synchronize()
        _check(out, torch.arange(n - rows + 1, n + 1, device="cuda"))


@pytest.mark.parametrize("dim", [64, 128])
def test_prompt(dim):
    from libosmos_amd import attn
    n, heads = 5000, 2
    q, k, v = (torch.zeros((n, h, dim), dtype=torch.float16, device="cuda") for h in (heads, 1, 1))
    q[..., 0], k[1:, :, 0], v[1:] = 1.0, LOW, 1.0
    out = torch.empty((n, heads, dim), device="cuda")
    print("small, prompt", dim, flush=True)
    attn.PromptAttention(q, k, v, _ints([0, n]), n, out, scale=1.0).run()
    torch.cuda.synchronize()
    _check(out, torch.arange(1, n + 1, device="cuda"))
