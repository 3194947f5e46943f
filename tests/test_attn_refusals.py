"""What the paged cache's and the attention's entry points refuse, before anything is queued (so on the CPU): shapes,
types, alignments and missing tables out of their contract (include/osmos_attn.h)."""
import ctypes

import pytest

from libosmos_amd import capi

A = 1 << 20  # a 16-byte aligned stand-in for an address: refused calls read nothing
P = ctypes.c_void_p


def _kv(**o):
    d = dict(data=A, scale=None, type=1, layers=2, pages=10, page=16, heads=2, dim=64)
    d.update(o)
    return capi.OsmosKv(**d)


def _step(**o):
    d = dict(start=A, len=A, table=A, seq=None, n_seq=2, n_tok=2, max_tok=1, max_len=100, seqs=2, table_stride=8)
    d.update(o)
    return capi.OsmosKvStep(**d)


def _attn(**o):
    d = dict(q=A, out=A, lse=None, q_stride=256, q_head=64, out_stride=256, out_head=64, q_type=1, out_type=1, heads=4,
             window=0, scale=0.125)
    d.update(o)
    return capi.OsmosAttn(**d)


def _rows(**o):
    d = dict(k=A, v=A, k_stride=128, k_head=64, v_stride=128, v_head=64, type=1, heads=2, dim=64)
    d.update(o)
    return capi.OsmosKvRows(**d)


BAD_KV = [dict(type=0), dict(type=2), dict(layers=0), dict(pages=0), dict(page=0), dict(page=24), dict(page=8192),
          dict(heads=0), dict(dim=0), dict(dim=24), dict(dim=272), dict(heads=4096, page=4096)]
BAD_CACHE = BAD_KV + [dict(data=None), dict(data=A + 8), dict(scale=A)]
BAD_STEP = [dict(start=None), dict(len=None), dict(table=None), dict(n_seq=0), dict(n_tok=0), dict(max_tok=0),
            dict(max_len=0), dict(seqs=1), dict(table_stride=0)]
BAD_ATTN = [dict(q=None), dict(out=None), dict(q=A + 8), dict(out=A + 2), dict(q_type=2), dict(out_type=0x200),
            dict(heads=0), dict(heads=3), dict(q_stride=257), dict(q_head=4), dict(out_stride=2), dict(scale=float("nan"))]


def _token(L, kv=None, step=None, attn=None, layer=0, name="osmos_attn_token"):
    return getattr(L, name)(ctypes.byref(attn or _attn()), ctypes.byref(kv or _kv()), layer, ctypes.byref(step or _step()),
                            P(A), 1 << 40, None)


@pytest.fixture(scope="module")
def L():
    return capi.lib()


@pytest.mark.parametrize("o", BAD_KV, ids=str)
def test_sizes(L, o):
    assert L.osmos_kv_bytes(ctypes.byref(_kv(**o))) == 0 and L.osmos_kv_scratch(ctypes.byref(_kv(**o))) == 0


def test_bytes(L):
    assert L.osmos_kv_bytes(ctypes.byref(_kv())) == 2 * 2 * 10 * 2 * 16 * 64 * 2
    assert L.osmos_kv_bytes(ctypes.byref(_kv(type=0x200, pages=1 << 20, heads=8, dim=256))) == 2 * 2 * (1 << 20) * 8 * 16 * 256


@pytest.mark.parametrize("o", BAD_CACHE, ids=str)
def test_cache(L, o):
    kv, st = ctypes.byref(_kv(**o)), ctypes.byref(_step())
    pool = ctypes.byref(capi.OsmosKvPool(A, A, A, A, 2, 8))
    assert not L.osmos_kv_append(kv, 0, st, 1, P(A), 128, P(A), 128, None)
    assert not _token(L, kv=_kv(**o)) and not _token(L, kv=_kv(**o), name="osmos_attn_chunk")
    assert not L.osmos_kv_grow(kv, pool, P(A), P(A), 1, None, None)
    assert not L.osmos_kv_fork(kv, pool, P(A), P(A), 1, None, None)
    assert not L.osmos_kv_free(kv, pool, P(A), 1, None)
    assert not L.osmos_kv_compact(kv, pool, None, None)
    assert not L.osmos_kv_copy(kv, P(A), P(A), 1, None)


@pytest.mark.parametrize("o", BAD_STEP, ids=str)
def test_step(L, o):
    assert not L.osmos_kv_append(ctypes.byref(_kv()), 0, ctypes.byref(_step(**o)), 1, P(A), 128, P(A), 128, None)
    assert not _token(L, step=_step(**o)) and not _token(L, step=_step(**o), name="osmos_attn_chunk")


@pytest.mark.parametrize("o", BAD_ATTN, ids=str)
def test_attn(L, o):
    assert not _token(L, attn=_attn(**o)) and not _token(L, attn=_attn(**o), name="osmos_attn_chunk")
    st = _step(len=None, table=None, seqs=0, table_stride=0, max_len=0)
    assert not L.osmos_attn_prompt(ctypes.byref(_attn(**o)), ctypes.byref(_rows()), ctypes.byref(st), P(A), 1 << 40, None)


@pytest.mark.parametrize("o", [dict(k=None), dict(v=A + 4), dict(k_stride=129), dict(v_head=60), dict(v_stride=1 << 25), dict(type=0), dict(type=0x200),
                               dict(heads=0), dict(dim=20), dict(dim=288)], ids=str)
def test_rows(L, o):
    st = _step(len=None, table=None, seqs=0, table_stride=0, max_len=0)
    assert not L.osmos_attn_prompt(ctypes.byref(_attn()), ctypes.byref(_rows(**o)), ctypes.byref(st), P(A), 1 << 40, None)


def test_others(L):
    kv, st = ctypes.byref(_kv()), ctypes.byref(_step())
    assert not _token(L, layer=2) and not _token(L, step=_step(max_tok=2))
    assert not L.osmos_kv_append(kv, 2, st, 1, P(A), 128, P(A), 128, None)
    assert not L.osmos_kv_append(kv, 0, st, 2, P(A), 128, P(A), 128, None)
    assert not L.osmos_kv_append(kv, 0, st, 1, P(A + 2), 128, P(A), 128, None)
    assert not L.osmos_kv_append(kv, 0, st, 1, P(A), 120, P(A), 128, None)
    assert not L.osmos_kv_append(kv, 0, st, 1, P(A), 128, P(A), 130, None)
    assert not L.osmos_kv_append(kv, 0, st, 1, None, 128, P(A), 128, None)
    for bad in (capi.OsmosKvPool(None, A, A, A, 2, 8), capi.OsmosKvPool(A + 4, A, A, A, 2, 8), capi.OsmosKvPool(A, None, A, A, 2, 8),
                capi.OsmosKvPool(A, A, None, A, 2, 8), capi.OsmosKvPool(A, A, A, None, 2, 8), capi.OsmosKvPool(A, A, A, A + 8, 2, 8),
                capi.OsmosKvPool(A, A, A, A, 0, 8), capi.OsmosKvPool(A, A, A, A, 2, 0)):
        assert not L.osmos_kv_compact(kv, ctypes.byref(bad), None, None)
        assert not L.osmos_kv_grow(kv, ctypes.byref(bad), P(A), P(A), 1, None, None)
    good = ctypes.byref(capi.OsmosKvPool(A, A, A, A, 2, 8))
    for n in (0, 1025):
        assert not L.osmos_kv_grow(kv, good, P(A), P(A), n, None, None)
        assert not L.osmos_kv_fork(kv, good, P(A), P(A), n, None, None)
        assert not L.osmos_kv_free(kv, good, P(A), n, None)
    assert not L.osmos_kv_copy(kv, P(A), P(A), 0, None)


def test_token_tiles(L):
    """a step whose tiles of 32 keys would pass 32 bits, by its bounds and by its tables' room"""
    assert not _token(L, step=_step(n_seq=66, seqs=66, max_len=0x7FFF0000, table_stride=1 << 27))
    assert not _token(L, step=_step(n_seq=1 << 20, seqs=1 << 20, max_len=0x7FFF0000, table_stride=1 << 13))
