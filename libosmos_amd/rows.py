"""The rows between a decoder block's products and the choice of the next token, for Python callers (include/osmos_rows.h):
torch tensors are the memory, each call one call of the C ABI on the given stream. As in attn.py the objects bind a call to its
buffers once, and a program runs them every step, eagerly or under graph capture; nothing here computes.

Streams: as attn.py's - a call is queued on the hipStream_t given as `stream`, the null stream for None; the buffers lie on the
device that is current when the object is made, and the calls are made with it current. What an object allocates (a table, a workspace)
lives as long as the object; calls that share one run in order on one stream.
"""
import ctypes

from . import attn, capi

HALVES, PAIRS = 0, 1


def _on_device(tensors):
    import torch
    index = torch.cuda.current_device()
    for t in tensors:
        if t is not None and (not t.is_cuda or t.device.index != index):
            raise ValueError("a tensor on another device than the current one (%s, cuda:%d)" % (t.device, index))
    return index


class _Call(attn._Call):
    """one call of the C ABI, made on the device of its buffers"""

    def _bind(self, *args, keep=()):
        import torch
        super()._bind(*args, keep=keep)
        self._device, self._current = _on_device([t for t in keep if isinstance(t, torch.Tensor)]), torch.cuda.current_device

    def run(self, stream=None):
        if self._current() != self._device:
            raise RuntimeError("%s: its buffers are on cuda:%d, which is not current" % (self.name, self._device))
        super().run(stream)


def _matrix(t, name, shape=None):
    """a (rows, dim) view's address and row stride"""
    if t.dim() != 2 or (t.shape[1] > 1 and t.stride(1) != 1) or not t.is_cuda:
        raise TypeError("%s: a device tensor (rows, dim) with contiguous dims is wanted" % name)
    if shape is not None and tuple(t.shape) != tuple(shape):
        raise ValueError("%s: %s is wanted" % (name, tuple(shape)))
    return t.data_ptr(), t.stride(0)


def _flat(t, name, dtype, count):
    if t.dtype != dtype or t.numel() != count or not t.is_contiguous() or not t.is_cuda:
        raise TypeError("%s: a contiguous %s device tensor of %d values is wanted" % (name, dtype, count))
    return t.data_ptr()


class Norm(_Call):
    """The root-mean-square norm of x's rows, of x + add where there is one (osmos_norm): y = x / sqrt(mean(x^2) + eps) (weight +
    offset). Into any of: sum, x + add of x's type (it may be x or add); out, rows; x16, mm's tiles (float16, whole tiles of 16 rows)
    with overflow, an int32 that a value past float16's range sets; codes and scales, q8_round's (int8 rows x dim, float32
    rows x dim / 32)."""
    name = "osmos_norm"

    def __init__(self, x, *, add=None, sum=None, weight=None, out=None, x16=None, overflow=None, codes=None, scales=None, eps=1e-6,
                 offset=0.0):
        import torch
        n, dim = x.shape if x.dim() == 2 else (0, 0)
        xp, xs = _matrix(x, "x")
        d = capi.OsmosNorm(x=xp, x_stride=xs, type=attn._type(x), n=n, dim=dim, eps=eps, offset=offset)
        for t, name in ((add, "add"), (sum, "sum")):
            if t is not None:
                if t.dtype != x.dtype:
                    raise TypeError("Norm: %s is of x's type" % name)
                p, s = _matrix(t, name, x.shape)
                setattr(d, name, p)
                setattr(d, name + "_stride", s)
        if weight is not None:
            d.weight, d.weight_type = _flat(weight, "weight", weight.dtype, dim), attn._type(weight)
        if out is not None:
            d.out, d.out_stride = _matrix(out, "out", x.shape)
            d.out_type = attn._type(out)
        if x16 is not None:
            d.x16 = _flat(x16, "x16", torch.float16, (n + 15) // 16 * 16 * dim)
            if overflow is None:
                raise ValueError("Norm: overflow is wanted with x16")
            d.overflow = _flat(overflow, "overflow", torch.int32, 1)
        if (codes is None) != (scales is None):
            raise ValueError("Norm: codes and scales come together")
        if codes is not None:
            d.codes, d.scales = _flat(codes, "codes", torch.int8, n * dim), _flat(scales, "scales", torch.float32, n * dim // 32)
        self.desc = d
        self._bind(ctypes.byref(d), keep=(x, add, sum, weight, out, x16, overflow, codes, scales))


class RopeTable:
    """The turns a token of each of rot / 2 pairs (osmos_rope_turns), on the device. scaling: None, or a dict with `kind` "linear",
    "ntk" (factor), "yarn" (factor, context, fast, slow) or "bands" (factor, context, low, high)."""
    KINDS = {"linear": 1, "ntk": 2, "yarn": 3, "bands": 4}

    def __init__(self, rot, base=10000.0, scaling=None):
        import torch
        s = dict(scaling or {})
        kind = s.pop("kind", None)
        if kind is not None and kind not in self.KINDS:
            raise ValueError("RopeTable: no scaling %r" % (kind,))
        wants = {None: (), "linear": ("factor",), "ntk": ("factor",), "yarn": ("factor", "context", "fast", "slow"),
                 "bands": ("factor", "context", "low", "high")}[kind]
        if set(s) != set(wants):
            raise ValueError("RopeTable: scaling %s takes %s" % (kind, ", ".join(wants)))
        d = capi.OsmosRopeScaling(self.KINDS.get(kind, 0), base, s.get("factor", 1.0), s.get("context", 1.0),
                                  s.get("low", s.get("slow", 0.0)), s.get("high", s.get("fast", 0.0)))
        turns, scale = (ctypes.c_double * max(1, rot // 2))(), ctypes.c_float()
        if not capi.lib().osmos_rope_turns(ctypes.byref(d), rot, turns, ctypes.byref(scale)):
            raise ValueError("osmos_rope_turns refused")
        self.rot, self.scale = rot, scale.value
        self.turns = torch.tensor(list(turns), dtype=torch.float64).cuda()


class _Rope(_Call):
    def _desc(self, table, q, out, k, k_out, pairs, q_weight, k_weight, eps, offset):
        import torch
        (qp, qs, qh), (op, os, oh) = attn._rows(q, "q"), attn._rows(out, "out")
        if q.shape != out.shape:
            raise ValueError("%s: q and out are (rows, heads, dim)" % type(self).__name__)
        n, heads, dim = q.shape
        d = capi.OsmosRope(turns=table.turns.data_ptr(), q=qp, q_stride=qs, q_head=qh, q_out=op, q_out_stride=os, q_out_head=oh,
                           type=attn._type(q), out_type=attn._type(out), heads=heads, n=n, dim=dim, rot=table.rot,
                           layout=PAIRS if pairs else HALVES, scale=table.scale, eps=eps, offset=offset)
        if k is not None:
            if k.dim() != 3 or k.shape[0] != n or k.shape[2] != dim or k.dtype != q.dtype:
                raise ValueError("%s: k is (q's rows, heads, q's dim) of q's type" % type(self).__name__)
            d.k, d.k_stride, d.k_head = attn._rows(k, "k")
            d.kv_heads = k.shape[1]
        if k_out is not None:
            if k is None or k_out.shape != k.shape or k_out.dtype != out.dtype:
                raise ValueError("%s: k_out is k's shape, of out's type" % type(self).__name__)
            d.k_out, d.k_out_stride, d.k_out_head = attn._rows(k_out, "k_out")
        for w, name in ((q_weight, "q_weight"), (k_weight, "k_weight")):
            if w is not None:
                setattr(d, name, _flat(w, name, torch.float32, dim))
        self.desc = d
        return ctypes.byref(d)


class Rope(_Rope):
    """q's (and k's) heads turned to the positions `pos` (int32, one a row) into out (and k_out), which may be q and k themselves.
    q_weight, k_weight: each head normed first (Norm's formula). pairs: neighbouring values turn together, not the halves'."""
    name = "osmos_rope"

    def __init__(self, table, pos, q, out, k=None, k_out=None, *, pairs=False, q_weight=None, k_weight=None, eps=1e-6, offset=0.0):
        if (k is None) != (k_out is None):
            raise ValueError("Rope: k and k_out come together")
        d = self._desc(table, q, out, k, k_out, pairs, q_weight, k_weight, eps, offset)
        if attn._ints(pos, "pos").numel() != q.shape[0]:
            raise ValueError("Rope: a position a row")
        self._bind(d, capi.addr(pos), keep=(table.turns, pos, q, out, k, k_out, q_weight, k_weight))


class RopeAppend(_Rope):
    """attn.Append with the step's rows turned to their places on the way: q into out (it may be q itself), k turned and v as it is
    into the layer's pages"""
    name = "osmos_rope_append"

    def __init__(self, table, cache, layer, step, q, out, k, v, *, pairs=False, q_weight=None, k_weight=None, eps=1e-6, offset=0.0):
        if tuple(k.shape) != (step.n_tok, cache.heads, cache.dim) or k.shape != v.shape or k.dtype != v.dtype:
            raise ValueError("RopeAppend: k and v are (rows, heads, dim) of one type, as the cache's")
        d = self._desc(table, q, out, k, None, pairs, q_weight, k_weight, eps, offset)
        vp, vs, vh = attn._rows(v, "v")
        self._bind(d, ctypes.byref(cache.desc), layer, ctypes.byref(step.desc), ctypes.c_void_p(vp), vs, vh,
                   keep=(table.turns, cache.data, cache.scale, step.start, step.len, step.table, step.seq, step.live, q, out, k, v, q_weight,
                         k_weight, cache, step))


class Sample(_Call):
    """One token for each row of logits (rows, vocab) by the given numbers u, 0 <= u < 1 (osmos_sample): token int32 (rows). A row's
    temperature, top_p, min_p (float32) and top_k (int32), where there are any. prob: the token's part of the kept
    weights; kept: how many tokens those are; probs (rows, vocab): every token's part."""
    name = "osmos_sample"

    def __init__(self, logits, u, token, *, temperature=None, top_k=None, top_p=None, min_p=None, prob=None, kept=None, probs=None):
        import torch
        lp, ls = _matrix(logits, "logits")
        n, vocab = logits.shape
        d = capi.OsmosSample(logits=lp, stride=ls, type=attn._type(logits), n=n, vocab=vocab)
        for t, name, dtype in ((u, "u", torch.float32), (token, "token", torch.int32), (temperature, "temperature", torch.float32),
                               (top_k, "top_k", torch.int32), (top_p, "top_p", torch.float32), (min_p, "min_p", torch.float32),
                               (prob, "prob", torch.float32), (kept, "kept", torch.int32)):
            if t is not None:
                setattr(d, name, _flat(t, name, dtype, n))
        if probs is not None:
            if tuple(probs.shape) != (n, vocab):
                raise ValueError("Sample: probs is (rows, vocab)")
            d.probs = _flat(probs, "probs", torch.float32, n * vocab)
        self.desc = d
        _on_device((logits,))
        nbytes = capi.lib().osmos_sample_workspace(ctypes.byref(d))
        self.workspace = torch.empty(nbytes, dtype=torch.uint8, device="cuda") if nbytes else None
        self._bind(ctypes.byref(d), capi.addr(self.workspace), nbytes,
                   keep=(logits, u, token, temperature, top_k, top_p, min_p, prob, kept, probs, self.workspace))
