"""A decoder block's attention over quantized projections, for Python callers: the query, key, value and output matrices in
GGUF row layout (mm_run), the step's keys and values into the paged cache (osmos_kv_append), attention over the cache
(osmos_attn_token for a step of single tokens, osmos_attn_chunk for prompts), with the norm before them and the rotary positions
between (rows.py); and a model's end, the last norm, the output matrix and the choice of tokens. What follows the attention in a block
is layer.LaneLayer (the routed experts). Rows are float32 as the library's products have them; a layer keeps one set of buffers, of
its longest step, that all its steps use: they are ordered on one stream, and a second stream takes a layer object of its
own. Nothing here computes.
"""
import ctypes

from . import attn, capi
from . import rows as row_calls


class _Calls(tuple):
    """a step's (append, attention), with the layer and the buffers that they were made for"""


def _need(ok, what):
    if not ok:
        raise RuntimeError("%s refused" % what)


def _weight(norm, dim):
    import torch
    if norm is not None and (norm.dtype != torch.float32 or tuple(norm.shape) != (dim,) or not norm.is_contiguous() or not norm.is_cuda):
        raise TypeError("norm is a contiguous float32 device tensor of dim values")
    row_calls._on_device((norm,))
    return norm


def _tiles(norm, eps, x, add, x16, overflow, stream):
    """x's rows, normed where there is a weight (x + add kept in x first), as mm's tiles"""
    n, dim = x.shape
    if norm is None:
        if add is not None:
            raise ValueError("add goes with a norm")
        return _need(capi.lib().mm_x16(capi.addr(x), dim, n, dim, capi.addr(x16), capi.addr(overflow), stream), "mm_x16")
    d = capi.OsmosNorm(x=x.data_ptr(), add=None if add is None else add.data_ptr(), sum=None if add is None else x.data_ptr(),
                       weight=norm.data_ptr(), x16=x16.data_ptr(), overflow=overflow.data_ptr(), x_stride=dim, add_stride=dim,
                       sum_stride=dim, type=attn.F32, weight_type=attn.F32, n=n, dim=dim, eps=eps)
    _need(capi.lib().osmos_norm(ctypes.byref(d), stream), "osmos_norm")


def _check_rows(owner, named, shape, device):
    import torch
    if torch.cuda.current_device() != device.index:
        raise RuntimeError("%s.forward: its buffers are on %s, which is not current" % (owner, device))
    for t, name in named:
        if t is None:
            continue
        if t.dtype != torch.float32 or not t.is_contiguous() or not t.is_cuda:
            raise TypeError("%s.forward: %s is a contiguous float32 device tensor" % (owner, name))
        if tuple(t.shape) != shape:
            raise ValueError("%s.forward: %s is (rows of the step, dim)" % (owner, name))
        if t.device != device:
            raise ValueError("%s.forward: %s is on another device than the buffers (%s, %s)" % (owner, name, t.device, device))


class AttentionLayer:
    def __init__(self, cache, layer, heads, wq, wk, wv, wo, dim, *, rope=None, pairs=False, q_weight=None, k_weight=None, norm=None,
                 eps=1e-6):
        """cache: attn.KvCache; layer: its layer here; heads: query heads; wq, wk, wv, wo: (GGUF type, uint8 device tensor),
        rows heads x cache.dim (wq), cache.heads x cache.dim (wk, wv) of dim values, dim rows of heads x cache.dim (wo).
        overflow: an int32 device value, set to 1 by a step whose x or attention rows are past f16's range (they become
        infinities in the products) and left so for the caller to read and clear.
        rope: rows.RopeTable: the queries and keys are turned to their tokens' places, by halves or `pairs`, each head normed first
        where there is a q_weight or k_weight (cache.dim values). norm: the block's first norm's weight (dim values): forward's x
        is then the residual stream. eps: of these norms"""
        import torch
        self.cache, self.layer, self.heads, self.dim = cache, layer, heads, dim
        self.w, self.wo = ((wq, heads * cache.dim), (wk, cache.heads * cache.dim), (wv, cache.heads * cache.dim)), wo
        for (t, _), rows in self.w:
            if not capi.lib().mm_fits(t, rows, dim):
                raise ValueError("AttentionLayer: mm does not take %d x %d of type %d" % (rows, dim, t))
        if not capi.lib().mm_fits(wo[0], dim, heads * cache.dim):
            raise ValueError("AttentionLayer: mm does not take the output matrix")
        if rope is None and (pairs or q_weight is not None or k_weight is not None):
            raise ValueError("AttentionLayer: pairs, q_weight and k_weight go with rope")
        if rope is not None and rope.rot > cache.dim:
            raise ValueError("AttentionLayer: rope turns more values than a head has")
        self.rope, self.heads_norm = rope, dict(pairs=pairs, q_weight=q_weight, k_weight=k_weight, eps=eps)
        self.norm, self.eps = _weight(norm, dim), eps
        self.overflow = torch.zeros(1, dtype=torch.int32, device="cuda")
        self._made, self._rows = {}, 0

    def _buffers(self, n):
        """a step's rows of the one set of buffers, which the longest step so far made"""
        import torch
        hd, kv = self.cache.dim, self.cache.heads
        if n > self._rows:
            tiles = (n + 15) // 16 * 16
            # (o zeros: a row that belongs to no sequence of the step is not written)
            self._made = {"qkv": torch.empty((n, self.heads + 2 * kv, hd), device="cuda"),
                          "o": torch.zeros((n, self.heads, hd), device="cuda"),
                          "x16": torch.empty(tiles * self.dim, dtype=torch.float16, device="cuda"),
                          "o16": torch.empty(tiles * self.heads * hd, dtype=torch.float16, device="cuda")}
            self._rows = n
        b = dict(self._made, o=self._made["o"][:n])
        b["q"], b["k"], b["v"] = b["qkv"][:n].split([self.heads, kv, kv], 1)
        return b

    def calls(self, step):
        """the append and the attention of a step, bound to its rows of this layer's buffers (made once a KvStep)"""
        b = self._buffers(step.n_tok)
        kind = attn.TokenAttention if step.desc.max_tok == 1 else attn.ChunkAttention
        if self.rope is None:
            append = attn.Append(self.cache, self.layer, step, b["k"], b["v"])
        else:
            append = row_calls.RopeAppend(self.rope, self.cache, self.layer, step, b["q"], b["q"], b["k"], b["v"], **self.heads_norm)
        calls = _Calls((append, kind(self.cache, self.layer, step, b["q"], b["o"])))
        calls.owner, calls.buffers, calls.n = self, b, step.n_tok
        return calls

    def forward(self, x, calls, out, stream=None, between=None, add=None):
        """out (n, dim) = the block's attention of x (n, dim), contiguous float32, for the step that `calls` were made for. With
        the layer's norm x is the residual stream: x + add (the block before's output, where there is one) is kept in x, and its
        norm goes into the projections.
        between(q, k, v, stream): queues on the stream what the model does to the projections' rows, in place, before the keys
        and values go into the cache (biases; norms and positions that rope does not cover): float32 views (n, heads, cache.dim)"""
        if getattr(calls, "owner", None) is not self:
            raise ValueError("AttentionLayer.forward: calls of another layer")
        L, n, b, (append, attention) = capi.lib(), calls.n, calls.buffers, calls
        _check_rows("AttentionLayer", ((x, "x"), (out, "out"), (add, "add")), (n, self.dim), b["qkv"].device)
        _tiles(self.norm, self.eps, x, add, b["x16"], self.overflow, stream)
        stride = b["qkv"].stride(0)
        for ((t, w), rows), y in zip(self.w, (b["q"], b["k"], b["v"])):
            _need(L.mm_run(t, capi.addr(w), rows, self.dim, capi.addr(b["x16"]), n, ctypes.c_void_p(y.data_ptr()), stride,
                           stream), "mm_run")
        if between:
            between(b["q"], b["k"], b["v"], stream)
        append.run(stream)
        attention.run(stream)
        cols = self.heads * self.cache.dim
        _need(L.mm_x16(capi.addr(b["o"]), cols, n, cols, capi.addr(b["o16"]), capi.addr(self.overflow), stream), "mm_x16")
        _need(L.mm_run(self.wo[0], capi.addr(self.wo[1]), self.dim, cols, capi.addr(b["o16"]), n, capi.addr(out), self.dim,
                       stream), "mm_run")
        return out


class TokenHead:
    def __init__(self, w, vocab, dim, norm=None, eps=1e-6):
        """a model's end: w: (GGUF type, uint8 device tensor), the output matrix's vocab rows of dim values; norm: the last norm's weight
        (dim values), where x is the residual stream. overflow: as AttentionLayer's"""
        import torch
        if not capi.lib().mm_fits(w[0], vocab, dim):
            raise ValueError("TokenHead: mm does not take %d x %d of type %d" % (vocab, dim, w[0]))
        self.w, self.vocab, self.dim, self.norm, self.eps = w, vocab, dim, _weight(norm, dim), eps
        self.overflow = torch.zeros(1, dtype=torch.int32, device="cuda")
        self._made = None

    def calls(self, u, token, **limits):
        """a step's choice of token.numel() tokens, bound to its rows of this head's buffers: u, token and the limits and outputs of
        rows.Sample (made once for these)"""
        import torch
        n = token.numel()
        if self._made is None or n > self._made[1].shape[0]:
            self._made = (torch.empty((n + 15) // 16 * 16 * self.dim, dtype=torch.float16, device="cuda"),
                          torch.empty((n, self.vocab), device="cuda"))
        x16, logits = self._made
        calls = _Calls((row_calls.Sample(logits[:n], u, token, **limits),))
        calls.owner, calls.buffers, calls.n = self, (x16, logits[:n]), n
        return calls

    def forward(self, x, calls, stream=None, add=None):
        """one token for each row of x (n, dim), contiguous float32, into the calls' `token`; returns the rows of logits, float32 (n,
        vocab), which the next step overwrites. With the head's norm x + add is kept in x, as AttentionLayer.forward's"""
        if getattr(calls, "owner", None) is not self:
            raise ValueError("TokenHead.forward: calls of another head")
        (x16, logits), n = calls.buffers, calls.n
        _check_rows("TokenHead", ((x, "x"), (add, "add")), (n, self.dim), logits.device)
        _tiles(self.norm, self.eps, x, add, x16, self.overflow, stream)
        _need(capi.lib().mm_run(self.w[0], capi.addr(self.w[1]), self.vocab, self.dim, capi.addr(x16), n, capi.addr(logits), self.vocab,
                                stream), "mm_run")
        calls[0].run(stream)
        return logits
