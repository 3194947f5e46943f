"""The checks that the paged cache's and the attention's entry points make before they queue anything (libosmos_amd/csrc/attnhost.h,
which they call), by themselves: each accepts a good call and refuses it with any one thing wrong. (The entry points also
return false where no launch is possible, as without a GPU, so that their refusals alone prove nothing there.)"""
import ctypes
import os
import re

import pytest

from libosmos_amd import capi
from tests import attn_host

A = 1 << 20  # a 256-byte aligned stand-in for an address: nothing is read
ROOM = 1 << 40
P, U32, U64, B = ctypes.c_void_p, ctypes.c_uint32, ctypes.c_uint64, ctypes.c_bool


def _of(cls, d):
    return lambda **o: cls(**dict(d, **o))


KV = _of(capi.OsmosKv, dict(data=A, type=1, layers=2, pages=10, page=16, heads=2, dim=64))
STEP = _of(capi.OsmosKvStep, dict(start=A, len=A, table=A, n_seq=2, n_tok=2, max_tok=1, max_len=100, seqs=2, table_stride=8))
PACKED = _of(capi.OsmosKvStep, dict(start=A, n_seq=2, n_tok=2, max_tok=1))
ATTN = _of(capi.OsmosAttn, dict(q=A, out=A, q_stride=256, q_head=64, out_stride=256, out_head=64, q_type=1, out_type=1, heads=4,
                                scale=0.125))
ROWS = _of(capi.OsmosKvRows, dict(k=A, v=A, k_stride=128, k_head=64, v_stride=128, v_head=64, type=1, heads=2, dim=64))
POOL = _of(capi.OsmosKvPool, dict(ref=A, len=A, table=A, scratch=A, seqs=2, table_stride=8))

GOOD_KV = [dict(), dict(type=30), dict(type=0x200), dict(type=0x200, scale=A), dict(layers=4096), dict(pages=0x7FFFFFF0), dict(page=1),
           dict(page=4096), dict(dim=16), dict(dim=80), dict(dim=256), dict(data=A + 16)]
BAD_KV = [dict(type=0), dict(type=2), dict(layers=0), dict(layers=4097), dict(pages=0), dict(pages=0x7FFFFFF1), dict(page=0), dict(page=24),
          dict(page=8192), dict(heads=0), dict(heads=4098), dict(dim=0), dict(dim=24), dict(dim=272), dict(heads=4096, page=4096),
          dict(data=None), dict(data=A + 8), dict(scale=A)]
GOOD_STEP = [dict(), dict(seq=A), dict(seq=A, seqs=1), dict(live=A), dict(n_seq=1), dict(max_len=0x7FFF0000, table_stride=1 << 20),
             dict(n_seq=1 << 20, seqs=1 << 20)]
BAD_STEP = [dict(start=None), dict(len=None), dict(table=None), dict(n_seq=0), dict(n_seq=(1 << 20) + 1, seqs=1 << 30), dict(n_tok=0),
            dict(n_tok=1 << 31), dict(max_tok=0), dict(max_tok=1 << 31), dict(max_len=0), dict(max_len=0x7FFF0001), dict(seqs=0, seq=A),
            dict(seqs=1), dict(table_stride=0)]
GOOD_ATTN = [dict(), dict(lse=A), dict(q_type=0, out_type=0), dict(q_type=30, out_type=30), dict(heads=2), dict(heads=4096),
             dict(window=0x7FFFFFFF), dict(scale=-1.0), dict(scale=0.0)]
BAD_ATTN = [dict(q=None), dict(out=None), dict(q=A + 8), dict(out=A + 2), dict(q_type=2), dict(q_type=0x200), dict(out_type=0x200),
            dict(heads=0), dict(heads=3), dict(heads=4098), dict(q_stride=257), dict(q_head=4), dict(out_stride=2), dict(out_head=62),
            dict(q_type=0, q_stride=258), dict(window=1 << 31), dict(scale=float("nan"))]
GOOD_ROWS = [dict(), dict(type=30), dict(dim=256), dict(k_stride=1 << 24, v_stride=1 << 24)]
BAD_ROWS = [dict(k=None), dict(v=None), dict(k=A + 8), dict(v=A + 4), dict(k_stride=129), dict(v_stride=132), dict(k_head=60),
            dict(v_head=60), dict(k_stride=(1 << 24) + 8), dict(v_stride=1 << 25), dict(type=0), dict(type=0x200), dict(heads=0),
            dict(heads=4097), dict(dim=0), dict(dim=20), dict(dim=288)]
GOOD_POOL = [dict(), dict(seqs=0x7FFFFFFF)]
BAD_POOL = [dict(ref=None), dict(ref=A + 4), dict(len=None), dict(table=None), dict(scratch=None), dict(scratch=A + 8), dict(seqs=0),
            dict(seqs=1 << 31), dict(table_stride=0)]


@pytest.fixture(scope="module")
def host(tmp_path_factory):
    h = attn_host.build(tmp_path_factory.mktemp("attn_host"))
    for name in ("append", "requests", "pool", "copy", "prompt", "chunk", "token"):
        getattr(h, "host_" + name).restype = B
    return h


def _ref(x):
    return None if x is None else ctypes.byref(x)


def _append(h, kv=KV(), step=STEP(), layer=0, type=1, k=A, ks=128, v=A, vs=128):
    return h.host_append(_ref(kv), U32(layer), _ref(step), U32(type), P(k), U64(ks), P(v), U64(vs))


def _paged(h, name, attn=ATTN(), kv=KV(), step=STEP(), layer=0, ws=A, room=ROOM):
    return getattr(h, "host_" + name)(_ref(attn), _ref(kv), U32(layer), _ref(step), P(ws), U64(room))


def _prompt(h, attn=ATTN(), rows=ROWS(), step=PACKED(), ws=A, room=ROOM):
    return h.host_prompt(_ref(attn), _ref(rows), _ref(step), P(ws), U64(room))


def _pool(h, kv=KV(), pool=POOL(), a=A, b=A, n=1):
    return h.host_requests(_ref(kv), _ref(pool), P(a), P(b), U32(n))


def test_good_calls(host):
    """every variant that the contract allows is taken"""
    for o in GOOD_KV:
        dim = o.get("dim", 64)
        attn = dict(q_head=dim, out_head=dim)
        assert _append(host, kv=KV(**o), ks=2 * dim, vs=2 * dim), o
        assert _paged(host, "chunk", ATTN(**attn), KV(**o)) and _paged(host, "token", ATTN(**attn), KV(**o)), o
        assert _pool(host, kv=KV(**o)) and host.host_pool(_ref(KV(**o)), _ref(POOL())), o
        assert host.host_copy(_ref(KV(**o)), P(A), P(A), U32(1 << 31)), o
    for o in GOOD_STEP:
        assert _append(host, step=STEP(**o)), o
        assert _paged(host, "chunk", step=STEP(**o)) and _paged(host, "token", step=STEP(**o)), o
    for o in GOOD_ATTN:
        assert _paged(host, "chunk", ATTN(**o)) and _paged(host, "token", ATTN(**o)) and _prompt(host, ATTN(**o)), o
    for o in GOOD_ROWS:
        assert _prompt(host, rows=ROWS(**o)), o
    for o in GOOD_POOL:
        assert _pool(host, pool=POOL(**o)), o
    for t, row in ((0, 128), (1, 128), (30, 128)):
        assert _append(host, type=t, ks=row, vs=row)
    assert _append(host, step=STEP(n_seq=1, n_tok=1), ks=0, vs=8)  # (one row: its stride is never used)
    assert _pool(host, n=1024)


def test_bad_caches(host):
    for o in BAD_KV + [None]:
        kv = None if o is None else KV(**o)
        assert not _append(host, kv=kv), o
        assert not _paged(host, "chunk", kv=kv) and not _paged(host, "token", kv=kv), o
        assert not _pool(host, kv=kv) and not host.host_pool(_ref(kv), _ref(POOL())), o
        assert not host.host_copy(_ref(kv), P(A), P(A), U32(1)), o


def test_bad_steps(host):
    for o in BAD_STEP + [None]:
        st = None if o is None else STEP(**o)
        assert not _append(host, step=st), o
        assert not _paged(host, "chunk", step=st) and not _paged(host, "token", step=st), o
    for o in (dict(start=None), dict(n_seq=0), dict(n_tok=0), dict(max_tok=0)):
        assert not _prompt(host, step=PACKED(**o)), o
    assert not _prompt(host, step=None)


def test_bad_attention(host):
    for o in BAD_ATTN + [None]:
        a = None if o is None else ATTN(**o)
        assert not _paged(host, "chunk", a) and not _paged(host, "token", a) and not _prompt(host, a), o
    for o in BAD_ROWS + [None]:
        assert not _prompt(host, rows=None if o is None else ROWS(**o)), o


def test_bad_others(host):
    for o in (dict(layer=2), dict(type=2), dict(type=0x200), dict(k=None), dict(v=None), dict(k=A + 2), dict(v=A + 8), dict(ks=120),
              dict(vs=120), dict(ks=130), dict(vs=130), dict(type=0, ks=130)):
        assert not _append(host, **o), o
    for name in ("chunk", "token"):
        assert not _paged(host, name, layer=2)
    assert not _paged(host, "token", step=STEP(max_tok=2)) and _paged(host, "chunk", step=STEP(max_tok=2))
    for o in BAD_POOL + [None]:
        p = None if o is None else POOL(**o)
        assert not _pool(host, pool=p) and not host.host_pool(_ref(KV()), _ref(p)), o
    for o in (dict(a=None), dict(b=None), dict(n=0), dict(n=1025)):
        assert not _pool(host, **o), o
    for a, b, n in ((None, A, 1), (A, None, 1), (A, A, 0)):
        assert not host.host_copy(_ref(KV()), P(a), P(b), U32(n))


def test_workspaces(host):
    """what osmos_attn_workspace says is enough, a byte less, no address or one that is not 256-byte aligned is refused; where it says
    none, none is asked for"""
    for call, step in (("token", STEP(max_len=5000, table_stride=400)), ("chunk", STEP(max_len=5000, table_stride=400)),
                       ("prompt", PACKED(n_tok=3000, max_tok=3000))):
        run = (lambda **o: _prompt(host, step=step, **o)) if call == "prompt" else (lambda **o: _paged(host, call, step=step, **o))
        need = capi.lib().osmos_attn_workspace(_ref(ATTN()), 2, 64, _ref(step))
        assert need and run(room=need) and not run(ws=None, room=need) and not run(ws=A + 16, room=need) and not run(room=0), call
        low, high = 0, need  # (the call's own need: the greater of two for a token step)
        while high - low > 1:
            mid = (low + high) // 2
            low, high = (low, mid) if run(room=mid) else (mid, high)
        assert high == need or step.max_tok == 1, call
        assert not run(room=high - 1), call
    assert not capi.lib().osmos_attn_workspace(_ref(ATTN()), 2, 64, _ref(STEP()))
    assert _paged(host, "token", ws=None, room=0) and _paged(host, "chunk", ws=None, room=0) and _prompt(host, ws=None, room=0)


def test_launch_bounds(host):
    """steps past a launch's 2^31 workgroups, 2^31 rows of query heads, or 2^32 tiles of keys"""
    long = dict(max_len=0x7FFF0000, table_stride=1 << 27)
    assert _paged(host, "token", step=STEP(n_seq=64, seqs=64, **long)) and not _paged(host, "token", step=STEP(n_seq=65, seqs=65, **long))
    many = dict(n_seq=1 << 20, n_tok=1 << 20, seqs=1 << 20)
    assert _paged(host, "token", step=STEP(**many)) and not _paged(host, "token", ATTN(heads=2048), step=STEP(**many))
    kv = KV(heads=2048, page=1)
    assert not _paged(host, "token", ATTN(heads=2048), kv, STEP(**many))
    assert _paged(host, "chunk", step=STEP(n_tok=(1 << 30) - 1, max_tok=9)) and not _paged(host, "chunk", step=STEP(n_tok=1 << 30, max_tok=9))
    assert not _prompt(host, ATTN(heads=4096), ROWS(heads=4096), PACKED(n_tok=1 << 30, max_tok=9))


def test_entry_points_use_the_checks():
    """each entry point's first statement is its check"""
    csrc = os.path.join(attn_host.HERE, "..", "libosmos_amd", "csrc")
    text = "".join(open(os.path.join(csrc, f)).read() for f in ("kv.hip", "attn.hip"))
    checks = {"osmos_kv_append": "kv::append_ok", "osmos_kv_grow": "kv::requests_ok", "osmos_kv_fork": "kv::requests_ok",
              "osmos_kv_free": "kv::requests_ok", "osmos_kv_compact": "kv::pool_ok", "osmos_kv_copy": "kv::copy_ok",
              "osmos_attn_prompt": "attn::prompt_ok", "osmos_attn_chunk": "attn::chunk_ok", "osmos_attn_token": "attn::token_ok"}
    for name, check in checks.items():
        body = re.search(r"OSM_API bool %s\([^{]*\{\s*([^\n]*)" % name, text).group(1)
        assert body.startswith("if (!%s(" % check) and body.endswith("return false;"), name
