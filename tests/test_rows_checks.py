"""What the entry points of include/osmos_rows.h refuse, by their checks compiled alone (tests/rows_host_driver.cpp): a good call
beside the bad ones, since without a GPU a call that a lost check let through would return false all the same. And the turns of
longer contexts against their formulas."""
import ctypes
import math
import os
import subprocess

import pytest

from libosmos_amd import capi

HERE = os.path.dirname(os.path.abspath(__file__))
A = 1 << 20  # (a 16-byte aligned stand-in for an address: the checks read nothing)
NAN, INF = float("nan"), float("inf")
R = ctypes.byref


@pytest.fixture(scope="module")
def H(tmp_path_factory):
    lib = str(tmp_path_factory.mktemp("rows") / "rows_host.so")
    subprocess.run(["g++", "-O2", "-std=c++17", "-Wall", "-Werror", "-shared", "-fPIC", os.path.join(HERE, "rows_host_driver.cpp"),
                    "-o", lib], check=True)
    h = ctypes.CDLL(lib)
    for f in ("host_norm", "host_rope", "host_rope_append", "host_turns", "host_sample", "host_launches"):
        getattr(h, f).restype = ctypes.c_bool
    h.host_rope_append.argtypes = [ctypes.c_void_p, ctypes.c_void_p, ctypes.c_uint32, ctypes.c_void_p, ctypes.c_void_p, ctypes.c_uint64,
                                   ctypes.c_uint64]
    return h


def _norm(**o):
    d = dict(x=A, add=A, sum=A, weight=A, out=A, x16=A, overflow=A, codes=A, scales=A, x_stride=64, add_stride=64, sum_stride=64,
             out_stride=70, type=0, weight_type=0, out_type=1, n=3, dim=64, eps=1e-6, offset=0.0)
    d.update(o)
    return capi.OsmosNorm(**d)


GOOD_NORM = [dict(), dict(add=None, sum=None, weight=None, out=None, x16=None, overflow=None), dict(dim=33, x16=None, codes=None, scales=None),
             dict(n=1, x_stride=0, add_stride=0, sum_stride=0, out_stride=0), dict(type=30, x=A + 2, out=A + 2, sum=None, weight_type=1), dict(eps=0.0),
             dict(dim=65536, x_stride=65536, add_stride=65536, sum_stride=65536, out_stride=65536), dict(dim=48, codes=None, scales=None),
             dict(sum=A, x=A + 64, add=A + 128, sum_stride=80)]
BAD_NORM = [dict(x=None), dict(x=A + 2), dict(type=2), dict(type=0x200), dict(n=0), dict(dim=0), dict(dim=65537, x_stride=1 << 17),
            dict(x_stride=63), dict(add_stride=63), dict(sum_stride=63), dict(out_stride=63), dict(out_type=0x200), dict(out=A + 1),
            dict(weight_type=2), dict(weight=A + 2), dict(dim=40), dict(dim=48), dict(x16=A + 8), dict(overflow=None), dict(codes=A + 8),
            dict(scales=None), dict(codes=None), dict(sum=None, out=None, x16=None, codes=None, scales=None), dict(eps=-1e-6), dict(eps=NAN),
            dict(eps=INF), dict(offset=NAN), dict(offset=INF), dict(sum=A, x_stride=70, add=A + 64), dict(add=A, x=A + 64, add_stride=70)]


@pytest.mark.parametrize("o", GOOD_NORM, ids=str)
def test_norm_good(H, o):
    assert H.host_norm(R(_norm(**o)))


@pytest.mark.parametrize("o", BAD_NORM, ids=str)
def test_norm_bad(H, o):
    assert not H.host_norm(R(_norm(**o)))
    assert not capi.lib().osmos_norm(R(_norm(**o)), None)


def _rope(**o):
    d = dict(turns=A, q=A, k=A, q_out=A + 4096, k_out=A + 8192, q_stride=512, q_head=64, k_stride=512, k_head=64, q_out_stride=256,
             q_out_head=64, k_out_stride=128, k_out_head=64, type=0, out_type=1, heads=4, kv_heads=2, n=3, dim=64, rot=64, layout=0, scale=1.0,
             eps=1e-6, offset=0.0)
    d.update(o)
    return capi.OsmosRope(**d)


SAME = dict(q_out=A, out_type=0, q_out_stride=512)
GOOD_ROPE = [dict(), dict(kv_heads=0, k=None, k_out=None), dict(rot=2), dict(rot=22), dict(layout=1), SAME, dict(k_out=A, out_type=0, k_out_stride=512),
             dict(n=1, q_stride=3), dict(heads=1, q_head=0, q_out_head=0), dict(q_weight=A, k_weight=A + 4), dict(dim=256, rot=256, q_head=256,
                                                                                                                 k_head=256, q_out_head=256,
                                                                                                                 k_out_head=256, q_out_stride=1024,
                                                                                                                 k_out_stride=512)]
BAD_ROPE = [dict(turns=None), dict(turns=A + 4), dict(n=0), dict(dim=0), dict(dim=60), dict(dim=264), dict(rot=0), dict(rot=3), dict(rot=66),
            dict(layout=2), dict(type=2), dict(out_type=0x200), dict(heads=0), dict(heads=4097), dict(kv_heads=4097), dict(scale=NAN),
            dict(scale=INF), dict(eps=-1.0), dict(eps=NAN), dict(offset=INF), dict(q_weight=A + 2), dict(k_weight=A + 1), dict(q=None),
            dict(q=A + 8), dict(q_out=None), dict(q_out=A + 4), dict(k=None), dict(k=A + 8), dict(k_out=None), dict(q_stride=514),
            dict(q_head=66), dict(q_head=32), dict(q_stride=32), dict(k_head=32), dict(k_out_stride=32), dict(q_out_head=68),
            dict(SAME, out_type=1), dict(SAME, q_out_stride=256), dict(SAME, q_out_head=128), dict(k_out=A), dict(k_out=A, out_type=0)]


@pytest.mark.parametrize("o", GOOD_ROPE, ids=str)
def test_rope_good(H, o):
    assert H.host_rope(R(_rope(**o)))


@pytest.mark.parametrize("o", BAD_ROPE, ids=str)
def test_rope_bad(H, o):
    assert not H.host_rope(R(_rope(**o)))
    assert not capi.lib().osmos_rope(R(_rope(**o)), ctypes.c_void_p(A), None)


def _kv(**o):
    d = dict(data=A, scale=None, type=1, layers=2, pages=10, page=16, heads=2, dim=64)
    d.update(o)
    return capi.OsmosKv(**d)


def _step(**o):
    d = dict(start=A, len=A, table=A, seq=None, n_seq=2, n_tok=3, max_tok=2, max_len=100, seqs=2, table_stride=8)
    d.update(o)
    return capi.OsmosKvStep(**d)


GOOD_APPEND = [{}, dict(rope=dict(k_out=None)), dict(v_stride=64, v_head=192), dict(kv=dict(type=0x200, scale=A))]
BAD_APPEND = [dict(rope=o) for o in BAD_ROPE if not any(k.startswith("k_out") for k in o)] + [
    dict(rope=dict(n=2)), dict(rope=dict(kv_heads=0)), dict(rope=dict(kv_heads=3)), dict(kv=dict(dim=128)), dict(kv=dict(heads=4)),
    dict(kv=dict(data=None)), dict(kv=dict(page=24)), dict(kv=dict(type=0)), dict(kv=dict(scale=A)), dict(layer=2), dict(step=dict(n_tok=4)),
    dict(step=dict(start=None)), dict(step=dict(len=None)), dict(step=dict(table=None)), dict(step=dict(seqs=1)), dict(step=dict(max_len=0)),
    dict(v=None), dict(v=A + 8), dict(v_stride=130), dict(v_stride=32), dict(v_head=32), dict(v_head=66)]


def _append(f, o, *tail):
    return f(R(_rope(**o.get("rope", {}))), R(_kv(**o.get("kv", {}))), o.get("layer", 1), R(_step(**o.get("step", {}))),
             ctypes.c_void_p(o.get("v", A)), o.get("v_stride", 128), o.get("v_head", 64), *tail)


@pytest.mark.parametrize("o", GOOD_APPEND, ids=str)
def test_append_good(H, o):
    assert _append(H.host_rope_append, o)


@pytest.mark.parametrize("o", BAD_APPEND, ids=str)
def test_append_bad(H, o):
    assert not _append(H.host_rope_append, o)
    assert not _append(capi.lib().osmos_rope_append, o, None)


def _sample(**o):
    d = dict(logits=A, u=A, token=A, temperature=A, top_p=A, min_p=A, top_k=A, prob=A, kept=A, probs=A, stride=1000, type=0, n=3, vocab=1000)
    d.update(o)
    return capi.OsmosSample(**d)


GOOD_SAMPLE = [{}, dict(temperature=None, top_p=None, min_p=None, top_k=None, prob=None, kept=None, probs=None), dict(vocab=1, stride=1),
               dict(n=1, stride=0), dict(type=1, logits=A + 2), dict(type=30), dict(vocab=1 << 20, stride=1 << 20)]
BAD_SAMPLE = [dict(logits=None), dict(logits=A + 2), dict(u=None), dict(token=None), dict(type=0x200), dict(type=2), dict(n=0), dict(vocab=0),
              dict(n=1 << 23), dict(vocab=(1 << 20) + 1, stride=1 << 21), dict(stride=999), dict(u=A + 2), dict(token=A + 1), dict(temperature=A + 2),
              dict(top_p=A + 2), dict(min_p=A + 2), dict(top_k=A + 2), dict(prob=A + 2), dict(kept=A + 2), dict(probs=A + 2)]


@pytest.mark.parametrize("o", GOOD_SAMPLE, ids=str)
def test_sample_good(H, o):
    assert H.host_sample(R(_sample(**o)))


@pytest.mark.parametrize("o", BAD_SAMPLE, ids=str)
def test_sample_bad(H, o):
    assert not H.host_sample(R(_sample(**o)))
    assert not capi.lib().osmos_sample(R(_sample(**o)), None, 0, None)


def test_more_rows_than_a_launch_holds(H):
    """refused before anything is queued (2^32 threads and more)"""
    fits = lambda blocks, threads: H.host_launches(ctypes.c_uint64(blocks), ctypes.c_uint32(threads))  # noqa: E731
    assert fits(1, 1024) and fits(4194303, 1024) and not fits(4194304, 1024) and not fits(0, 64) and not fits(1 << 40, 64)
    n = 0x3FFFFFF
    assert not capi.lib().osmos_norm(R(_norm(n=1 << 30, dim=32, x_stride=32, add_stride=32, sum_stride=32, out_stride=32)), None)
    assert not capi.lib().osmos_rope(R(_rope(n=1 << 27, kv_heads=0)), ctypes.c_void_p(A), None)
    assert not capi.lib().osmos_sample(R(_sample(n=n >> 3, vocab=8, stride=8)), ctypes.c_void_p(A), 1 << 40, None)


def test_no_workspace(H):
    """a call that wants a workspace and is not given one"""
    d = _sample(n=1, vocab=1 << 20, stride=1 << 20)
    need = capi.lib().osmos_sample_workspace(R(d))
    for ws, size in ((None, need), (A, need - 1), (A + 64, need)):
        if need:
            assert not capi.lib().osmos_sample(R(d), ctypes.c_void_p(ws), size, None)
    assert capi.lib().osmos_sample_workspace(R(_sample(vocab=0))) == 0 and capi.lib().osmos_sample_workspace(None) == 0


def _turns(H, rot, kind=0, base=10000.0, factor=1.0, context=1.0, low=0.0, high=0.0):
    t, s = (ctypes.c_double * (rot // 2 + 1))(), ctypes.c_float(-1)
    d = capi.OsmosRopeScaling(kind, base, factor, context, low, high)
    return (list(t)[:rot // 2], s.value) if H.host_turns(R(d), rot, t, R(s)) else None


@pytest.mark.parametrize("rot", [2, 20, 64, 128, 256])
def test_turns(H, rot):
    plain, one = _turns(H, rot)
    assert one == 1.0
    for i, f in enumerate(plain):
        assert math.isclose(f, 10000.0 ** (-2 * i / rot) / (2 * math.pi), rel_tol=1e-14)
    linear, one = _turns(H, rot, 1, factor=4.0)
    assert one == 1.0 and all(math.isclose(a, b / 4, rel_tol=1e-14) for a, b in zip(linear, plain))
    if rot >= 4:
        ntk, one = _turns(H, rot, 2, factor=8.0)
        # the slowest pair turns `factor` times as slowly, the fastest as before
        assert one == 1.0 and ntk[0] == plain[0] and math.isclose(ntk[-1] * 8, plain[-1], rel_tol=1e-12)
    bands, one = _turns(H, rot, 4, factor=8.0, context=8192.0, low=1.0, high=4.0)
    assert one == 1.0
    for a, b in zip(bands, plain):
        n = 8192 * b
        want = b if n >= 4 else b / 8 if n <= 1 else b * (n - 1) / 3 + b / 8 * (1 - (n - 1) / 3)
        assert math.isclose(a, want, rel_tol=1e-13)
    yarn, scale = _turns(H, rot, 3, factor=16.0, context=8192.0, low=1.0, high=32.0)
    assert math.isclose(scale, 0.1 * math.log(16) + 1, rel_tol=1e-6)
    for i, (a, b) in enumerate(zip(yarn, plain)):
        n = 8192 * b
        assert b / 16 * (1 - 1e-13) <= a <= b * (1 + 1e-13)
        if n > 32 * 10000 ** (2 / rot):  # (a whole pair past the ramp's ends, which are whole pairs)
            assert math.isclose(a, b, rel_tol=1e-13)
        if n < 10000 ** (-2 / rot):
            assert math.isclose(a, b / 16, rel_tol=1e-13)
    assert all(x >= y for x, y in zip(yarn, yarn[1:]))


@pytest.mark.parametrize("rot,o", [(0, {}), (3, {}), (258, {}), (64, dict(kind=5)), (64, dict(base=1.0)), (64, dict(base=NAN)), (64, dict(base=INF)),
                                   (64, dict(kind=1, factor=0.5)), (64, dict(kind=1, factor=NAN)), (2, dict(kind=2, factor=2.0)),
                                   (64, dict(kind=3, factor=2.0, context=0.0, low=1.0, high=32.0)),
                                   (64, dict(kind=3, factor=2.0, context=8192.0, low=32.0, high=32.0)),
                                   (64, dict(kind=4, factor=2.0, context=8192.0, low=0.0, high=4.0)),
                                   (64, dict(kind=4, factor=2.0, context=8192.0, low=1.0, high=NAN))], ids=str)
def test_turns_refused(H, rot, o):
    assert _turns(H, rot, **o) is None
