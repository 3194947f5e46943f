"""A token step's keys cut into chunks (libosmos_amd/csrc/attnhost.h, which the kernel uses): never more chunks than the launch and its
workspace have room for, and every sequence's keys covered, up to steps of nearly 2^32 tiles of 32 keys, where an earlier rule's
chunk length wrapped."""
import ctypes
import random

import pytest

from libosmos_amd import capi
from tests import attn_host

MOST = 0x7FFF0000  # tokens a sequence may have


@pytest.fixture(scope="module")
def host(tmp_path_factory):
    return attn_host.build(tmp_path_factory.mktemp("attn_host"))


def _old_chunk(total, want):
    even = (total // want + 1) & 0xFFFFFFFF
    tiles32 = (even * 32) & 0xFFFFFFFF
    return 384 if tiles32 <= 384 else ((even + 3) // 4 * 128) & 0xFFFFFFFF


def _covers(chunk, groups, most, chunks_of):
    """groups: (sequences, keys of each); no sequence's count of chunks wraps, none needs a chunk more than there is room for"""
    if not 0 < chunk < 2 ** 31:
        return False
    total = 0
    for n, k in groups:
        c = chunks_of(k, chunk)
        if c * chunk < k or (c - 1) * chunk > max(k - 1, 0):
            return False
        total += n * c
    return total <= most


def _cases():
    rng = random.Random(1)
    for kv_heads, heads in ((1, 1), (1, 64), (2, 16), (8, 32), (32, 32), (64, 64), (512, 512), (4096, 4096)):
        for groups in ([(1, 1)], [(1, 333)], [(1, MOST)], [(31, MOST)], [(63, MOST)], [(2, MOST), (50, 1)], [(1 << 20, 1)],
                       [(1 << 20, 4094 * 32)], [(1 << 16, 65534 * 32)], [(200, 2 ** 29 - 64)], [(1, 0), (5, 385), (3, 384)]):
            yield kv_heads, heads, groups
        for _ in range(200):
            groups = [(rng.randint(1, 50), int(2 ** rng.uniform(0, 30.9))) for _ in range(rng.randint(1, 6))]
            n, longest = sum(g[0] for g in groups), max(g[1] for g in groups)
            if n * (longest // 32 + 1) <= 0xFFFFFFFF:  # (what the call takes)
                yield kv_heads, heads, groups


def test_chunks_fit_their_launch(host):
    host.host_chunk_keys.restype = host.host_chunks_of.restype = ctypes.c_uint32
    old_wrong = cases = 0
    for kv_heads, heads, groups in _cases():
        n, longest = sum(g[0] for g in groups), max(max(g[1] for g in groups), 1)
        assert n * (longest // 32 + 1) <= 0xFFFFFFFF
        st = capi.OsmosKvStep(None, None, None, None, n, n, 1, longest, n, 1)
        a = capi.OsmosAttn(heads=heads)
        want, most, split = (ctypes.c_uint32() for _ in range(3))
        host.host_cut(ctypes.byref(a), kv_heads, 128, ctypes.byref(st), *(ctypes.byref(x) for x in (want, most, split)))
        total = sum(m * (-(-k // 32)) for m, k in groups)
        chunk = host.host_chunk_keys(ctypes.c_uint32(total), want)
        count = lambda k, c: host.host_chunks_of(k, ctypes.c_uint32(c))  # noqa: E731
        assert _covers(chunk, groups, most.value, count), (kv_heads, heads, groups, chunk)
        assert split.value or all(count(k, chunk) == 1 for _, k in groups)
        old = _old_chunk(total, want.value)
        old_wrong += not _covers(old, groups, most.value, lambda k, c: 1 if k <= (c if c < 2 ** 31 else c - 2 ** 32) else (k + c - 1) // c if c else 0)
        if old < 2 ** 31 and total // want.value < (1 << 26) - 5:
            assert old == chunk
        cases += 1
    assert cases > 500 and old_wrong > 0  # (the old rule fails for some of these)
