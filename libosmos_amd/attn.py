"""The paged cache of keys and values and the attention over it, for Python callers (include/osmos_attn.h): torch tensors
are the memory, each call one call of the C ABI on the given stream. The objects bind a call to its buffers once - a
serving program makes them with its buffers and runs them every step, eagerly or under graph capture; nothing here
computes.

Streams: a call is queued on the hipStream_t given as `stream`, on the null stream for None - never on torch's current stream by
itself, so that inside torch.cuda.stream(s) s.cuda_stream is passed. What a call or a pool allocates (workspaces, scratch) comes from
torch's allocator for the stream current when the object is made and lives as long as the object: keep that until the work that
it queued elsewhere is done. Calls that share an object run in order on one stream.
"""
import ctypes

from . import capi

F32, F16, BF16, F8 = 0, 1, 30, 0x200


def _type(t):
    import torch
    types = {torch.float32: F32, torch.float16: F16, torch.bfloat16: BF16, torch.float8_e4m3fn: F8}
    if t.dtype not in types:
        raise TypeError("osmos attention: no type for %s" % t.dtype)
    return types[t.dtype]


def _ints(t, name):
    import torch
    if t.dtype != torch.int32 or not t.is_contiguous() or not t.is_cuda:
        raise TypeError("%s: a contiguous int32 device tensor is wanted" % name)
    return t


def _rows(t, name):
    """a (rows, heads, dim) view's address and strides: the innermost dimension contiguous"""
    if t.dim() != 3 or (t.shape[2] > 1 and t.stride(2) != 1) or not t.is_cuda:
        raise TypeError("%s: a device tensor (rows, heads, dim) with contiguous dims is wanted" % name)
    return t.data_ptr(), t.stride(0), t.stride(1)


class KvCache:
    """A cache over `data`, a device tensor (layers, 2, pages, heads, page, dim) of float16, bfloat16 or float8_e4m3fn;
    `scale` (float8): float32 (layers, 2, heads)."""

    def __init__(self, data, scale=None):
        import torch
        if data.dim() != 6 or data.shape[1] != 2 or not data.is_contiguous() or not data.is_cuda:
            raise TypeError("KvCache: a contiguous device tensor (layers, 2, pages, heads, page, dim) is wanted")
        layers, _, pages, heads, page, dim = data.shape
        if scale is not None and (scale.dtype != torch.float32 or tuple(scale.shape) != (layers, 2, heads) or
                                  not scale.is_contiguous() or not scale.is_cuda):
            raise TypeError("KvCache: scale is a contiguous float32 device tensor (layers, 2, heads)")
        self.data, self.scale = data, scale
        self.layers, self.pages, self.heads, self.page, self.dim = layers, pages, heads, page, dim
        self.desc = capi.OsmosKv(data.data_ptr(), None if scale is None else scale.data_ptr(), _type(data), layers, pages,
                                 page, heads, dim)
        if not capi.lib().osmos_kv_bytes(ctypes.byref(self.desc)):
            raise ValueError("KvCache: a shape out of range")

    @classmethod
    def empty(cls, dtype, layers, pages, heads, page, dim, scale=None):
        import torch
        return cls(torch.zeros((layers, 2, pages, heads, page, dim), dtype=dtype, device="cuda"), scale)

    def copy(self, src, dst, stream=None):
        """pages src[i] to pages dst[i] (int32 device tensors), in every layer"""
        if src.numel() != dst.numel():
            raise ValueError("KvCache.copy: as many pages to as from")
        if not capi.lib().osmos_kv_copy(ctypes.byref(self.desc), capi.addr(_ints(src, "src")), capi.addr(_ints(dst, "dst")),
                                        src.numel(), stream):
            raise RuntimeError("osmos_kv_copy refused")


class KvPool:
    """Which pages are whose: ref (pages), len (sequences), table (sequences, most pages), int32 device tensors."""

    def __init__(self, cache, ref, len, table):
        import torch
        if ref.numel() != cache.pages or table.dim() != 2 or table.shape[0] != len.numel():
            raise ValueError("KvPool: ref has a count a page, table a row a sequence")
        self.cache, self.ref, self.len, self.table = cache, ref, len, table
        for t, name in ((ref, "ref"), (len, "len"), (table, "table")):
            _ints(t, name)
        nbytes = capi.lib().osmos_kv_scratch(ctypes.byref(cache.desc))
        self.scratch = torch.empty(nbytes, dtype=torch.uint8, device="cuda")
        self.desc = capi.OsmosKvPool(ref.data_ptr(), len.data_ptr(), table.data_ptr(), self.scratch.data_ptr(),
                                     table.shape[0], table.shape[1])
        self._kv, self._pool = ctypes.byref(cache.desc), ctypes.byref(self.desc)

    @classmethod
    def empty(cls, cache, seqs, most):
        """no page in use: `seqs` sequences of at most `most` tokens"""
        import torch
        width = -(-most // cache.page)
        return cls(cache, torch.zeros(cache.pages, dtype=torch.int32, device="cuda"),
                   torch.zeros(seqs, dtype=torch.int32, device="cuda"),
                   torch.full((seqs, width), -1, dtype=torch.int32, device="cuda"))

    def grow(self, seq, add, done=None, stream=None):
        """add[i] more tokens for seq[i]; done[i] 0: refused. a step queued behind it takes `done` as its `live`"""
        if add.numel() != seq.numel() or (done is not None and done.numel() != seq.numel()):
            raise ValueError("KvPool.grow: seq, add and done have one entry a request")
        if not capi.lib().osmos_kv_grow(self._kv, self._pool, capi.addr(_ints(seq, "seq")), capi.addr(_ints(add, "add")),
                                        seq.numel(), capi.addr(done if done is None else _ints(done, "done")), stream):
            raise RuntimeError("osmos_kv_grow refused")

    def fork(self, src, dst, done=None, stream=None):
        if src.numel() != dst.numel() or (done is not None and done.numel() != src.numel()):
            raise ValueError("KvPool.fork: src, dst and done have one entry a request")
        if not capi.lib().osmos_kv_fork(self._kv, self._pool, capi.addr(_ints(src, "src")), capi.addr(_ints(dst, "dst")),
                                        src.numel(), capi.addr(done if done is None else _ints(done, "done")), stream):
            raise RuntimeError("osmos_kv_fork refused")

    def free(self, seq, stream=None):
        if not capi.lib().osmos_kv_free(self._kv, self._pool, capi.addr(_ints(seq, "seq")), seq.numel(), stream):
            raise RuntimeError("osmos_kv_free refused")

    def compact(self, live=None, stream=None):
        if not capi.lib().osmos_kv_compact(self._kv, self._pool, capi.addr(live if live is None else _ints(live, "live")),
                                           stream):
            raise RuntimeError("osmos_kv_compact refused")


class KvStep:
    """The rows of one step (OsmosKvStep): start (sequences + 1), len and table as the pool's, seq the step's sequences'
    places in them (None: in order). n_tok rows in all; no sequence brings more than max_tok, none is longer than max_len.
    live (None: all): 0 for a sequence that takes no part, KvPool.grow's `done` where the step follows it unread: its rows are
    not appended and attend to nothing."""

    def __init__(self, start, len=None, table=None, *, n_tok, max_tok, max_len=0, seq=None, live=None):
        self.start, self.len, self.table, self.seq, self.live = start, len, table, seq, live
        for t, name in ((start, "start"), (len, "len"), (table, "table"), (seq, "seq"), (live, "live")):
            if t is not None:
                _ints(t, name)
        if seq is not None and seq.numel() != start.numel() - 1:
            raise ValueError("KvStep: seq has an entry a sequence of the step")
        if live is not None and live.numel() != start.numel() - 1:
            raise ValueError("KvStep: live has an entry a sequence of the step")
        if table is not None and (table.dim() != 2 or len is None or table.shape[0] != len.numel()):
            raise ValueError("KvStep: table has a row a sequence of len")
        at = lambda t: None if t is None else t.data_ptr()  # noqa: E731
        self.n_tok = n_tok
        self.desc = capi.OsmosKvStep(at(start), at(len), at(table), at(seq), start.numel() - 1, n_tok, max_tok, max_len,
                                     0 if table is None else table.shape[0], 0 if table is None else table.shape[1],
                                     at(live))


class _Call:
    """One call of the C ABI bound to its buffers, which it keeps alive"""
    name = None

    def _bind(self, *args, keep=()):
        self._f, self._args, self._keep = getattr(capi.lib(), self.name), args, keep

    def run(self, stream=None):
        if not self._f(*self._args, stream):
            raise RuntimeError("%s refused" % self.name)


class Append(_Call):
    """the step's rows k, v (n_tok, heads, dim; contiguous rows) into a layer's pages"""
    name = "osmos_kv_append"

    def __init__(self, cache, layer, step, k, v):
        if tuple(k.shape) != (step.n_tok, cache.heads, cache.dim) or k.shape != v.shape or k.dtype != v.dtype:
            raise ValueError("Append: k and v are (rows, heads, dim) of one type")
        (kp, ks, kh), (vp, vs, vh) = _rows(k, "k"), _rows(v, "v")
        if (kh, vh) != (cache.dim, cache.dim) and cache.heads > 1:
            raise TypeError("Append: a row's heads lie one after another")
        self._bind(ctypes.byref(cache.desc), layer, ctypes.byref(step.desc), _type(k), ctypes.c_void_p(kp), ks,
                   ctypes.c_void_p(vp), vs, keep=(cache, step, k, v))


class _Attention(_Call):
    def _attn(self, step, q, out, lse, heads, dim, window, scale):
        import torch
        if tuple(q.shape[::2]) != (step.n_tok, dim) or q.shape != out.shape or q.shape[1] % heads:
            raise ValueError("%s: q and out are (rows, heads, dim), heads a multiple of the keys'" % type(self).__name__)
        if lse is not None and (lse.dtype != torch.float32 or tuple(lse.shape) != tuple(q.shape[:2]) or
                                not lse.is_contiguous() or not lse.is_cuda):
            raise TypeError("lse is a contiguous float32 device tensor (rows, heads)")
        (qp, qs, qh), (op, os, oh) = _rows(q, "q"), _rows(out, "out")
        self.desc = capi.OsmosAttn(qp, op, None if lse is None else lse.data_ptr(), qs, qh, os, oh, _type(q), _type(out),
                                   q.shape[1], window, dim ** -0.5 if scale is None else scale)
        nbytes = capi.lib().osmos_attn_workspace(ctypes.byref(self.desc), heads, dim, ctypes.byref(step.desc))
        ws = torch.empty(nbytes, dtype=torch.uint8, device="cuda") if nbytes else None
        self.workspace = ws
        return ctypes.byref(self.desc), ctypes.byref(step.desc), capi.addr(ws), nbytes


class PromptAttention(_Attention):
    """whole prompts: packed rows q, k, v, sequence s the rows start[s] .. start[s + 1] - 1, none longer than `longest`"""
    name = "osmos_attn_prompt"

    def __init__(self, q, k, v, start, longest, out, lse=None, window=0, scale=None):
        if k.shape != v.shape or k.dtype != v.dtype or k.shape[0] != q.shape[0]:
            raise ValueError("PromptAttention: k and v are (rows, heads, dim) of one type, a row each of q's")
        step = KvStep(start, n_tok=q.shape[0], max_tok=longest)
        a, st, ws, nbytes = self._attn(step, q, out, lse, k.shape[1], k.shape[2], window, scale)
        (kp, ks, kh), (vp, vs, vh) = _rows(k, "k"), _rows(v, "v")
        self.rows = capi.OsmosKvRows(kp, vp, ks, kh, vs, vh, _type(k), k.shape[1], k.shape[2])
        self._bind(a, ctypes.byref(self.rows), st, ws, nbytes, keep=(q, k, v, start, out, lse, step))


class ChunkAttention(_Attention):
    """the step's rows over a layer's pages, where their own keys and values already are"""
    name = "osmos_attn_chunk"

    def __init__(self, cache, layer, step, q, out, lse=None, window=0, scale=None):
        a, st, ws, nbytes = self._attn(step, q, out, lse, cache.heads, cache.dim, window, scale)
        self._bind(a, ctypes.byref(cache.desc), layer, st, ws, nbytes, keep=(cache, step, q, out, lse))


class TokenAttention(ChunkAttention):
    """ChunkAttention where every sequence brings one row"""
    name = "osmos_attn_token"
