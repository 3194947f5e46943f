"""A decoder block's attention over quantized projections, for Python callers: the query, key, value and output matrices in
GGUF row layout (mm_run), the step's keys and values into the paged cache (osmos_kv_append), attention over the cache
(osmos_attn_token for a step of single tokens, osmos_attn_chunk for prompts). What follows it in a block is
layer.LaneLayer (the routed experts). Rows are float32 as the library's products have them; a layer keeps one set of buffers, of
its longest step, that all its steps use: they are ordered on one stream, and a second stream takes a layer object of its
own. Nothing here computes.
"""
import ctypes

from . import attn, capi


class _Calls(tuple):
    """a step's (append, attention), with the layer and the buffers that they were made for"""


class AttentionLayer:
    def __init__(self, cache, layer, heads, wq, wk, wv, wo, dim):
        """cache: attn.KvCache; layer: its layer here; heads: query heads; wq, wk, wv, wo: (GGUF type, uint8 device tensor),
        rows heads x cache.dim (wq), cache.heads x cache.dim (wk, wv) of dim values, dim rows of heads x cache.dim (wo).
        overflow: an int32 device value, set to 1 by a step whose x or attention rows are past f16's range (they become
        infinities in the products) and left so for the caller to read and clear"""
        import torch
        self.cache, self.layer, self.heads, self.dim = cache, layer, heads, dim
        self.w, self.wo = ((wq, heads * cache.dim), (wk, cache.heads * cache.dim), (wv, cache.heads * cache.dim)), wo
        for (t, _), rows in self.w:
            if not capi.lib().mm_fits(t, rows, dim):
                raise ValueError("AttentionLayer: mm does not take %d x %d of type %d" % (rows, dim, t))
        if not capi.lib().mm_fits(wo[0], dim, heads * cache.dim):
            raise ValueError("AttentionLayer: mm does not take the output matrix")
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
        calls = _Calls((attn.Append(self.cache, self.layer, step, b["k"], b["v"]),
                        kind(self.cache, self.layer, step, b["q"], b["o"])))
        calls.owner, calls.buffers, calls.n = self, b, step.n_tok
        return calls

    def forward(self, x, calls, out, stream=None, between=None):
        """out (n, dim) = the block's attention of x (n, dim), contiguous float32, for the step that `calls` were made for.
        between(q, k, v, stream): queues on the stream what the model does to the projections' rows, in place, before the keys
        and values go into the cache (rotary positions, norms, biases): float32 views (n, heads, cache.dim)"""
        import torch
        if getattr(calls, "owner", None) is not self:
            raise ValueError("AttentionLayer.forward: calls of another layer")
        for t, name in ((x, "x"), (out, "out")):
            if t.dtype != torch.float32 or not t.is_contiguous() or not t.is_cuda:
                raise TypeError("AttentionLayer.forward: %s is a contiguous float32 device tensor" % name)
            if tuple(t.shape) != (calls.n, self.dim):
                raise ValueError("AttentionLayer.forward: %s is (rows of the step, dim)" % name)
        L, n, b, (append, attention) = capi.lib(), calls.n, calls.buffers, calls

        def need(ok, what):
            if not ok:
                raise RuntimeError("%s refused" % what)
        need(L.mm_x16(capi.addr(x), self.dim, n, self.dim, capi.addr(b["x16"]), capi.addr(self.overflow), stream), "mm_x16")
        stride = b["qkv"].stride(0)
        for ((t, w), rows), y in zip(self.w, (b["q"], b["k"], b["v"])):
            need(L.mm_run(t, capi.addr(w), rows, self.dim, capi.addr(b["x16"]), n, ctypes.c_void_p(y.data_ptr()), stride,
                          stream), "mm_run")
        if between:
            between(b["q"], b["k"], b["v"], stream)
        append.run(stream)
        attention.run(stream)
        cols = self.heads * self.cache.dim
        need(L.mm_x16(capi.addr(b["o"]), cols, n, cols, capi.addr(b["o16"]), capi.addr(self.overflow), stream), "mm_x16")
        need(L.mm_run(self.wo[0], capi.addr(self.wo[1]), self.dim, cols, capi.addr(b["o16"]), n, capi.addr(out), self.dim,
                      stream), "mm_run")
        return out
