"""A paged cache of keys and values over torch tensors, for serving a causal LUT-NN transformer on one MI355X.

The reference recomputes whole sequences in every forward (inference-engine/src/host/transformer_layer.cpp:211-230) and has no
cache; this is what a caller needs to feed a model its new tokens only.  Everything stays on the device, the bookkeeping included: once a cache is made no
call here waits for the GPU, and a step (reserve, then per layer append and attend) can be recorded into a HIP graph.

    cache = PagedCache(ctx, pimdl, layers=12, pages=4096, kv_heads=12, head_dim=64, page_tokens=16, dtype="f16", seqs=64, max_len=2048)
    cache.reserve(seqs, counts)                      # room for counts[i] more positions of sequence seqs[i]
    for layer in ...:
        cache.append(layer, k, v, starts, seqs)      # the new tokens' keys and values, packed: row b owns starts[b] .. starts[b + 1] - 1
        cache.attend(layer, q, out, starts, heads, seqs)
"""
import ctypes
import math

import torch

_TORCH = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
_CODES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}


class PagedCache:
    """k, v: [layers][pages][kv_heads][page_tokens][head_dim]; tables int32 [seqs][width], lengths int32 [seqs], refs int32 [pages]
    (see pimdl_page_book).  `lacking` (int32 [1], on the device) tells how many pages the last reserve or fork was short of: 0 means done,
    -1 that a sequence would outgrow its row of the table; nothing else has changed then, and append writes nothing until a later reserve or
    fork has had enough."""

    def __init__(self, ctx, pimdl, layers, pages, kv_heads, head_dim, page_tokens=16, dtype="f16", seqs=64, max_len=4096):
        dev = torch.device("cuda", torch.cuda.current_device())
        shape = (layers, pages, kv_heads, page_tokens, head_dim)
        k, v = (torch.zeros(shape, device=dev, dtype=_TORCH[dtype]) for _ in range(2))
        tables = torch.full((seqs, -(-max_len // page_tokens)), -1, device=dev, dtype=torch.int32)
        self._bind(ctx, pimdl, k, v, tables, torch.zeros(seqs, device=dev, dtype=torch.int32), torch.zeros(pages, device=dev, dtype=torch.int32))

    @classmethod
    def over(cls, ctx, pimdl, k, v, tables, lengths, refs):
        """A cache over tensors that exist already; they stay the caller's."""
        self = cls.__new__(cls)
        self._bind(ctx, pimdl, k, v, tables, lengths, refs)
        return self

    def _bind(self, ctx, pimdl, k, v, tables, lengths, refs):
        if k.dim() != 5 or k.shape != v.shape or k.dtype != v.dtype or k.dtype not in _CODES:
            raise ValueError("k and v must be [layers][pages][kv_heads][page_tokens][head_dim] of one type: float32, float16 or bfloat16")
        layers, pages, kv_heads, page_tokens, head_dim = k.shape
        if tables.dim() != 2 or lengths.shape != tables.shape[:1] or refs.shape != (pages,):
            raise ValueError("tables must be [seqs][width], lengths [seqs] and refs [pages]")
        if any(t.dtype != torch.int32 for t in (tables, lengths, refs)):
            raise ValueError("tables, lengths and refs must be int32")
        if not all(t.is_cuda and t.device == k.device and t.is_contiguous() for t in (k, v, tables, lengths, refs)):
            raise ValueError("a cache's tensors must be contiguous and on one GPU")
        self.ctx, self.k, self.v, self.tables, self.lengths, self.refs = ctx, k, v, tables, lengths, refs
        self.lacking = torch.zeros(1, device=k.device, dtype=torch.int32)
        # torch has queued zeros on its own stream, the context may have another: they are there when this returns (under a capture, from the replay on)
        if not torch.cuda.is_current_stream_capturing():
            torch.cuda.current_stream(k.device).synchronize()
        self.layers, self.kv_heads, self.head_dim, self.page_tokens = layers, kv_heads, head_dim, page_tokens
        self._lib = pimdl.lib()
        self._unlimited = pimdl.UNLIMITED
        layer_bytes = k[0].numel() * k.element_size() if layers else 0
        self._layer = [pimdl.PagedCacheDesc(k.data_ptr() + i * layer_bytes, v.data_ptr() + i * layer_bytes, tables.data_ptr(), lengths.data_ptr(),
                                            self.lacking.data_ptr(), pages, page_tokens, kv_heads, head_dim, tables.shape[0], tables.shape[1], _CODES[k.dtype]) for i in range(layers)]
        self._pools = (ctypes.c_void_p * 2)(k.data_ptr(), v.data_ptr())
        self._book = pimdl.PageBook(tables.data_ptr(), lengths.data_ptr(), refs.data_ptr(), self.lacking.data_ptr(), tables.shape[0], tables.shape[1], pages,
                                    page_tokens, ctypes.cast(self._pools, ctypes.POINTER(ctypes.c_void_p)), 2, layers, layer_bytes // max(pages, 1))

    def _list(self, t, name):
        if t.dtype != torch.int32 or t.dim() != 1 or not t.is_contiguous():
            raise ValueError(f"{name} must be a contiguous int32 vector")
        return t.data_ptr(), t.shape[0]

    def _rows(self, t, columns, name):
        """Address, row stride and type of a packed tensor; a column range of a wider one is fine."""
        if t.dim() != 2 or t.shape[1] != columns or (t.shape[1] > 1 and t.stride(1) != 1) or t.dtype not in _CODES:
            raise ValueError(f"{name} must be [tokens][{columns}] with unit column stride")
        stride = t.stride(0) if t.shape[0] > 1 else columns  # (of a single row it says nothing)
        if stride > self._unlimited:
            raise ValueError(f"{name}: a row stride of {stride} (up to 2^32 - 1)")
        return t.data_ptr(), stride, _CODES[t.dtype]

    def _batch(self, starts, seqs):
        at, n = self._list(starts, "starts")
        if n < 1:
            raise ValueError("starts must hold one number more than there are sequences")
        if seqs is None:
            return None, at, n - 1
        to, m = self._list(seqs, "seqs")
        if m != n - 1:
            raise ValueError("starts must hold one number more than seqs")
        return to, at, m

    def _of(self, layer):
        if not 0 <= layer < self.layers:
            raise IndexError(f"a cache of {self.layers} layers has no layer {layer}")
        return self._layer[layer]

    def check_batch(self, starts, seqs=None):
        """Refuses tensors that append and attend would not take for a batch."""
        _, _, batch = self._batch(starts, seqs)
        if seqs is None and batch > self.tables.shape[0]:
            raise ValueError(f"{batch} rows: the cache has {self.tables.shape[0]} sequences")

    def append(self, layer, k, v, starts, seqs=None):
        """New tokens' keys and values [tokens][kv_heads * head_dim] into the last positions of their sequences (whose room `reserve` has made)."""
        if k.shape != v.shape or k.stride() != v.stride() or k.dtype != v.dtype:
            raise ValueError("k and v must have one shape, stride and type")
        ka, ks, kt = self._rows(k, self.kv_heads * self.head_dim, "k")
        to, at, batch = self._batch(starts, seqs)
        self.ctx._check(self._lib.pimdl_cache_append(self.ctx._h, self._of(layer), to, at, batch, k.shape[0], ka, v.data_ptr(), ks, kt))

    def attend(self, layer, q, out, starts, heads, seqs=None, left=None, sinks=0, scale=None):
        """Causal attention of the new tokens (q, out: [tokens][heads * head_dim]) over everything that their sequences have in the cache, or, with
        `left`, over the `left` positions before each of them and the first `sinks`."""
        columns = heads * self.head_dim
        if q.shape != out.shape or q.dtype != out.dtype:
            raise ValueError("q and out must have one shape and type")
        qa, qs, qt = self._rows(q, columns, "q")
        oa, os_, _ = self._rows(out, columns, "out")
        left = self._unlimited if left is None else left
        if not (0 <= left <= self._unlimited and 0 <= sinks <= self._unlimited):
            raise ValueError(f"left={left} and sinks={sinks} must be counts of positions, below 2^32")
        to, at, batch = self._batch(starts, seqs)
        self.ctx._check(self._lib.pimdl_attention_paged(self.ctx._h, self._of(layer), to, at, batch, q.shape[0], qa, oa, heads, qs, os_, qt,
                                                        left, sinks,
                                                        1.0 / math.sqrt(self.head_dim) if scale is None else scale))

    def reserve(self, seqs, counts):
        """Makes sequence seqs[i] counts[i] positions longer (pages: the lowest free ones)."""
        a, n = self._list(seqs, "seqs")
        c, m = self._list(counts, "counts")
        if n != m:
            raise ValueError("seqs and counts must have one length")
        self.ctx._check(self._lib.pimdl_pages_reserve(self.ctx._h, self._book, a, c, n))

    def fork(self, parents, children):
        """Gives each empty sequence children[i] what parents[i] has: whole pages are shared, a partly filled last one is copied."""
        a, n = self._list(parents, "parents")
        c, m = self._list(children, "children")
        if n != m:
            raise ValueError("parents and children must have one length")
        self.ctx._check(self._lib.pimdl_pages_fork(self.ctx._h, self._book, a, c, n))

    def free(self, seqs):
        """Empties the sequences and gives their pages back."""
        a, n = self._list(seqs, "seqs")
        self.ctx._check(self._lib.pimdl_pages_free(self.ctx._h, self._book, a, n))

    def compact(self):
        """Moves all pages in use to the front of the cache."""
        self.ctx._check(self._lib.pimdl_pages_compact(self.ctx._h, self._book))

    def copy(self, src, dst):
        """Copies page src[i] to page dst[i] in every layer."""
        a, n = self._list(src, "src")
        c, m = self._list(dst, "dst")
        if n != m:
            raise ValueError("src and dst must have one length")
        self.ctx._check(self._lib.pimdl_pages_copy(self.ctx._h, self._book, a, c, n))
