"""The paged cache's pages: rows written into them (osmos_kv_append) bit for bit against a host restatement, and the
pool's operations (osmos_kv_grow, _fork, _free, _compact, _copy) against a plain sequential model of them."""
import random

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

T = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32, "f8": torch.float8_e4m3fn}


def _ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def _bits(t):
    return t.contiguous().view(torch.uint8).cpu()


@pytest.mark.parametrize("src", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("kind", ["f16", "bf16", "f8"])
@pytest.mark.parametrize("heads,dim,page,rows,lens", [
    (1, 16, 1, [1], [1]), (8, 128, 16, [1, 1, 1], [1, 16, 300]), (3, 80, 32, [40, 0, 7], [40, 9, 100]),
    (2, 256, 8, [5, 20], [3, 21]), (5, 96, 64, [70], [200]), (4, 64, 16, [1] * 70, list(range(1, 71)))])
def test_append(src, kind, heads, dim, page, rows, lens):
    from libosmos_amd import attn
    g = torch.Generator(device="cuda")
    g.manual_seed(dim)
    layers, n = 2, sum(rows)
    need = [-(-m // page) for m in lens]
    pages, width = sum(need) + 2, max(need) + 1
    order = torch.randperm(pages, generator=g, device="cuda").int()
    table = torch.full((len(lens), width), -1, dtype=torch.int32, device="cuda")
    at = 0
    for i, m in enumerate(need):
        table[i, :m] = order[at:at + m]
        at += m
    if len(rows) > 2:
        table[0, 0] = pages + 5  # (a page that does not exist: its rows are dropped)
    scale = None if kind != "f8" else 0.01 + torch.rand((layers, 2, heads), generator=g, device="cuda")
    data = torch.full((layers, 2, pages, heads, page, dim), 3.0, device="cuda").to(T[kind])
    fused = torch.randn((n, 2 * heads * dim + 64), generator=g, device="cuda") * 3
    fused.view(-1)[::97] *= 300.0
    fused.view(-1)[5::501] = float("nan")
    fused.view(-1)[7::777] = float("inf")
    fused = fused.to(T[src])
    k, v = fused[:, :heads * dim].view(n, heads, dim), fused[:, heads * dim:2 * heads * dim].view(n, heads, dim)
    starts = [0]
    for r in rows:
        starts.append(starts[-1] + r)
    want = data.clone()
    raw = want.view(torch.uint8) if kind == "f8" else want
    for i, (r, m) in enumerate(zip(rows, lens)):
        for j in range(r):
            pos = m - r + j
            if pos < 0 or not 0 <= int(table[i, pos // page]) < pages:
                continue
            for w, x in enumerate((k, v)):
                y = x[starts[i] + j].float()
                if kind == "f8":
                    y = (y / scale[1, w][:, None]).clamp(-448, 448)
                y = y.to(T[kind])
                raw[1, w, table[i, pos // page], :, pos % page] = y.view(torch.uint8) if kind == "f8" else y
    step = attn.KvStep(_ints(starts), _ints(lens), table, n_tok=n, max_tok=max(rows), max_len=max(lens))
    print("append", src, kind, heads, dim, page, flush=True)
    attn.Append(attn.KvCache(data, scale), 1, step, k, v).run()
    torch.cuda.synchronize()
    got, want = data.float(), want.float()
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    assert torch.equal(got.nan_to_num(9.0, 8.0, -8.0), want.nan_to_num(9.0, 8.0, -8.0))


def test_append_quotients():
    """8-bit values are the quotients' own roundings: every float16 value over scales of many sizes, those next to a rounding's
    edge among them"""
    from libosmos_amd import attn
    heads, dim, page = 64, 128, 8
    bits = torch.arange(65536, device="cuda").to(torch.int32)
    x = bits.to(torch.int16).view(torch.float16).view(8, heads, dim)
    scale = torch.empty((1, 2, heads), device="cuda")
    for seed, (low, high) in enumerate(((0.001, 0.02), (0.5, 1.5), (1e-22, 1e-17), (1e18, 1e21), (-0.3, -0.01))):
        scale.uniform_(low, high, generator=torch.Generator("cuda").manual_seed(seed))
        data = torch.zeros((1, 2, 1, heads, page, dim), device="cuda").to(T["f8"])
        step = attn.KvStep(_ints([0, 8]), _ints([8]), _ints([[0]]), n_tok=8, max_tok=8, max_len=8)
        k, v = x, x.flip(0).contiguous()
        print("quotients", low, flush=True)
        attn.Append(attn.KvCache(data, scale), 0, step, k, v).run()
        torch.cuda.synchronize()
        for w, t in enumerate((k, v)):
            want = (t.float() / scale[0, w][:, None]).clamp(-448, 448).to(T["f8"]).float().transpose(0, 1)
            got = data[0, w, 0].float()
            assert torch.equal(torch.isnan(got), torch.isnan(want))
            assert torch.equal(got.nan_to_num(9.0), want.nan_to_num(9.0)), (low, w)


class Model:
    """the pool, one request after another"""

    def __init__(self, pages, page, seqs, width):
        self.ref, self.len, self.page, self.width = [0] * pages, [0] * seqs, page, width
        self.table = [[-1] * width for _ in range(seqs)]

    def used(self, s):
        return -(-self.len[s] // self.page)

    def grow(self, seq, add):
        """(granted, the copies made)"""
        start_ref = list(self.ref)
        free = [p for p, r in enumerate(start_ref) if r == 0]
        done, copies, stopped, taken = [], [], False, {}
        for i, (s, a) in enumerate(zip(seq, add)):
            ok = 0 <= s < len(self.len) and s not in seq[:i] and a >= 0 and self.len[s] + a <= self.width * self.page
            if not ok:
                done.append(0)
                continue
            have, now = self.used(s), -(-(self.len[s] + a) // self.page)
            last = self.table[s][have - 1] if a and self.len[s] % self.page else None
            copy = last is not None and start_ref[last] - taken.get(last, 0) > 1
            if last is not None:
                taken[last] = taken.get(last, 0) + 1
            need = now - have + copy
            if stopped or need > len(free):
                stopped = True
                done.append(0)
                continue
            got, free = free[:need], free[need:]
            if copy:
                copies.append((last, got[0]))
                self.ref[last] -= 1
                self.table[s][have - 1] = got[0]
            for j, p in enumerate(got[copy:]):
                self.table[s][have + j] = p
            for p in got:
                self.ref[p] = 1
            self.len[s] += a
            done.append(1)
        return done, copies

    def fork(self, src, dst):
        done = []
        before = list(self.len)
        for i, (a, b) in enumerate(zip(src, dst)):
            n = len(self.len)
            ok = 0 <= a < n and 0 <= b < n and a not in dst and b not in dst[:i] and before[b] == 0
            done.append(int(ok))
            if ok:
                self.len[b], self.table[b] = self.len[a], [p if j < self.used(a) else -1 for j, p in enumerate(self.table[a])]
                for p in self.table[b][:self.used(b)]:
                    self.ref[p] += 1
        return done

    def free(self, seq):
        for s in seq:
            if 0 <= s < len(self.len):
                for j in range(self.used(s)):
                    self.ref[self.table[s][j]] -= 1
                    self.table[s][j] = -1
                self.len[s] = 0

    def compact(self):
        live = sum(r > 0 for r in self.ref)
        holes = [p for p in range(live) if self.ref[p] == 0]
        move = [p for p in range(live, len(self.ref)) if self.ref[p] > 0]
        to = dict(zip(move, holes))
        for a, b in to.items():
            self.ref[b], self.ref[a] = self.ref[a], 0
        for s in range(len(self.len)):
            for j in range(self.used(s)):
                self.table[s][j] = to.get(self.table[s][j], self.table[s][j])
        return live, list(to.items())


@pytest.mark.parametrize("pages,page,seqs,width,heads,dim,layers", [
    (40, 16, 12, 9, 2, 64, 1), (1, 8, 3, 4, 1, 16, 2), (700, 4, 60, 30, 1, 16, 1), (40000, 1, 200, 700, 1, 16, 1),
    (333, 32, 20, 40, 3, 80, 3)])
@pytest.mark.parametrize("kind", ["f16", "f8"])
def test_pool(pages, page, seqs, width, heads, dim, layers, kind):
    """a random history of growing, forking, freeing and compacting: counts, lengths, tables, outcomes and the pages'
    contents after each step"""
    from libosmos_amd import attn
    rng = random.Random(pages)
    raw = torch.randint(0, 120, (layers, 2, pages, heads, page, dim), dtype=torch.uint8, device="cuda")
    data = raw.view(T["f8"]) if kind == "f8" else raw.to(T["f16"])
    raw = data.view(torch.uint8)
    cache = attn.KvCache(data)
    pool = attn.KvPool.empty(cache, seqs, width * page)
    m = Model(pages, page, seqs, width)

    def same(what):
        torch.cuda.synchronize()
        assert pool.ref.tolist() == m.ref, what
        assert pool.len.tolist() == m.len, what
        assert pool.table.tolist() == m.table, what

    for turn in range(14):
        what = rng.choice(("grow", "grow", "grow", "fork", "free", "compact"))
        n = rng.randint(1, max(1, seqs // 2))
        print("pool", pages, kind, turn, what, n, flush=True)
        if what == "grow":
            seq = [rng.randrange(-1, seqs + 1) for _ in range(n)]
            add = [rng.choice((0, 1, 1, page, rng.randint(0, width * page // 2), -1)) for _ in range(n)]
            done = _ints([5] * n)
            before = raw.clone()
            pool.grow(_ints(seq), _ints(add), done)
            want, copies = m.grow(seq, add)
            same(what)
            assert done.tolist() == want
            for a, b in copies:
                before[:, :, b] = before[:, :, a]
            assert torch.equal(raw, before)
        elif what == "fork":
            src, dst = [rng.randrange(-1, seqs) for _ in range(n)], [rng.randrange(-1, seqs + 1) for _ in range(n)]
            done = _ints([5] * n)
            pool.fork(_ints(src), _ints(dst), done)
            want = m.fork(src, dst)
            same(what)
            assert done.tolist() == want
        elif what == "free":
            seq = [rng.randrange(-1, seqs + 1) for _ in range(n)]
            pool.free(_ints(seq))
            m.free(seq)
            same(what)
        else:
            live, before = _ints([-1]), raw.clone()
            pool.compact(live)
            n_live, moves = m.compact()
            same(what)
            assert int(live) == n_live
            for a, b in moves:
                before[:, :, b] = before[:, :, a]
            assert torch.equal(raw, before)


def test_forked_page_copied_once_each():
    """four holders of a partly filled page that all grow: three copies, the last holder keeps the page"""
    from libosmos_amd import attn
    data = torch.randn((2, 2, 10, 2, 16, 64), device="cuda").half()
    cache = attn.KvCache(data)
    pool = attn.KvPool.empty(cache, 4, 64)
    pool.grow(_ints([0]), _ints([20]))
    pool.fork(_ints([0, 0, 0]), _ints([1, 2, 3]))
    torch.cuda.synchronize()
    assert pool.ref.tolist() == [4, 4] + [0] * 8
    before = data.clone()
    print("four holders", flush=True)
    pool.grow(_ints([2, 0, 3, 1]), _ints([1, 1, 1, 1]))
    torch.cuda.synchronize()
    assert pool.ref.tolist() == [4, 1, 1, 1, 1] + [0] * 5
    assert [r[:2] for r in pool.table.tolist()] == [[0, 3], [0, 1], [0, 2], [0, 4]]
    for p in (2, 3, 4):
        assert torch.equal(data[:, :, p], before[:, :, 1])
    assert torch.equal(data[:, :, :2], before[:, :, :2]) and torch.equal(data[:, :, 5:], before[:, :, 5:])


@pytest.mark.parametrize("page,heads,dim,kind", [(1, 1, 16, "f8"), (16, 8, 128, "bf16"), (64, 3, 80, "f16"), (4096, 2, 256, "f16")])
def test_copy(page, heads, dim, kind):
    from libosmos_amd import attn
    raw = torch.randint(0, 120, (2, 2, 12, heads, page, dim), dtype=torch.uint8, device="cuda")
    data = raw.view(T["f8"]) if kind == "f8" else raw.to(T[kind])
    want = data.view(torch.uint8).clone()
    src, dst = [0, 5, 5, -1, 3], [1, 7, 11, 2, 12]
    for a, b in zip(src[:3], dst[:3]):
        want[:, :, b] = want[:, :, a]
    print("copy", page, heads, dim, kind, flush=True)
    attn.KvCache(data).copy(_ints(src), _ints(dst))
    torch.cuda.synchronize()
    assert torch.equal(data.view(torch.uint8), want)
