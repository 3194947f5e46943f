"""osmos_kv_append where a row has fewer 16-byte pieces than a wave has lanes (few kv heads: multi-query models, a kv head a
GPU) and the step more sequences than the row has pieces: every row lands, bit for bit."""
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


def _ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("seqs", [1, 33, 64, 65, 200, 4500])
@pytest.mark.parametrize("heads,dim", [(1, 16), (1, 64), (1, 128), (2, 64), (3, 80), (2, 96), (1, 256)])
def test_every_sequence_of_a_step(heads, dim, seqs):
    """one row a sequence, and in turn 0 .. 3 rows a sequence"""
    from libosmos_amd import attn
    g = torch.Generator(device="cuda")
    g.manual_seed(seqs + dim)
    page, width = 16, 3
    for rows in ([1] * seqs, [(i * 7 + 1) % 4 for i in range(seqs)]):
        lens = [r + (i * 5) % 40 for i, r in enumerate(rows)]
        n, pages = sum(rows), seqs * width
        table = torch.randperm(pages, generator=g, device="cuda").int().view(seqs, width)
        data = torch.full((1, 2, pages, heads, page, dim), 3.0, dtype=torch.float16, device="cuda")
        k, v = (torch.randn((n, heads, dim), generator=g, device="cuda").half() for _ in range(2))
        starts = [0]
        for r in rows:
            starts.append(starts[-1] + r)
        owner = torch.repeat_interleave(torch.arange(seqs), torch.tensor(rows)).cuda()
        pos = torch.tensor([m - r + j for r, m in zip(rows, lens) for j in range(r)], device="cuda")
        want = data.clone()
        for w, x in enumerate((k, v)):
            want[0, w][table[owner, pos // page].long(), :, pos % page] = x
        step = attn.KvStep(_ints(starts), _ints(lens), table, n_tok=n, max_tok=max(rows), max_len=max(lens))
        print("append", heads, dim, seqs, n, flush=True)
        attn.Append(attn.KvCache(data), 0, step, k, v).run()
        torch.cuda.synchronize()
        lost = sum(not torch.equal(data[0, w][table[owner[t], pos[t] // page].long(), :, pos[t] % page], x[t])
                   for w, x in enumerate((k, v)) for t in range(n)) if not torch.equal(data, want) else 0
        assert torch.equal(data, want), "%d of %d rows' keys or values lost" % (lost, 2 * n)
