"""A paged cache of keys and values over torch tensors, for serving a causal LUT-NN transformer on one MI355X.

The reference recomputes whole sequences in every forward (inference-engine/src/host/transformer_layer.cpp:211-230) and has no
cache; this is what a caller needs to feed a model its new tokens only.  Everything stays on the device, the bookkeeping included: once a cache is made no
call here waits for the GPU (but see DraftTree.order), and a step (reserve, then per layer append and attend) can be recorded into a HIP graph.

    cache = PagedCache(ctx, pimdl, layers=12, pages=4096, kv_heads=12, head_dim=64, page_tokens=16, dtype="f16", seqs=64, max_len=2048)
    cache.reserve(seqs, counts)                      # room for counts[i] more positions of sequence seqs[i]
    for layer in ...:
        cache.append(layer, k, v, starts, seqs)      # the new tokens' keys and values, packed: row b owns starts[b] .. starts[b + 1] - 1
        cache.attend(layer, q, out, starts, heads, seqs)

Rotated positions: a Rotary turns the keys on their way into the cache, and the queries along with them:

    rotary = Rotary(ctx, pimdl, head_dim=64, base=10000.0)
        cache.append(layer, k, v, starts, seqs, rotary=rotary, q=q, q_out=q)

Drafts: the new tokens of a sequence may be a tree of candidates.  A step over them reserves room for all, and ends with the branch that the model agrees with:

    tree = DraftTree(ctx, pimdl, tokens, most=64)    # room for so many tokens, in trees of up to 64
    tree.build(parents, starts)                      # parents[t]: the node (of its own sequence's) that token t follows, -1: none
        cache.append(layer, k, v, starts, seqs, rotary=rotary, q=q, q_out=q, tree=tree)
        cache.attend(layer, q, out, starts, heads, seqs, tree=tree)
    cache.accept(tree, last, kept, starts, seqs)     # last[b]: the node that the branch of row b ends with
"""
import ctypes
import math
import weakref

import torch

_TORCH = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
_CODES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}


def _int_list(t, name):
    if t.dtype != torch.int32 or t.dim() != 1 or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous int32 vector")
    return t.data_ptr(), t.shape[0]


def _packed(t, columns, name):
    """Address, row stride and type of a packed tensor; a column range of a wider one is fine."""
    shape, stride, dtype = t.shape, t.stride(), _CODES.get(t.dtype)
    if len(shape) != 2 or shape[1] != columns or (columns > 1 and stride[1] != 1) or dtype is None:
        raise ValueError(f"{name} must be [tokens][{columns}] with unit column stride")
    stride = stride[0] if shape[0] > 1 else columns  # (of a single row it says nothing)
    if stride > 0xFFFFFFFF:
        raise ValueError(f"{name}: a row stride of {stride} (up to 2^32 - 1)")
    return t.data_ptr(), stride, dtype


class Rotary:
    """Turns queries and keys by their positions: at position p the pair (a, b) of a head's columns that belongs to frequency f becomes
    (a cos pf - b sin pf, a sin pf + b cos pf).  The first `dims` columns of a head turn (all of them by default), column i with i + dims / 2 (pairs="halves") or 2 i with
    2 i + 1 ("neighbours").  Frequency i is base^(-2 i / dims), or freqs[i] (float64 [dims / 2] on the device, radians a position): scaled ones for
    longer contexts, say.  A position times a frequency is below 2^52 (positions below 2^31: frequencies up to 2^21, a base of 2^-21 or more)."""

    def __init__(self, ctx, pimdl, head_dim, base=10000.0, dims=None, pairs="halves", freqs=None):
        if pairs not in pimdl.PAIRS:
            raise ValueError(f"pairs={pairs!r}: 'halves' or 'neighbours'")
        if freqs is None:
            dims = head_dim if dims is None else dims
            if dims % 2 or not 2 <= dims <= head_dim:
                raise ValueError(f"dims={dims} must be even, 2 .. head_dim={head_dim}")
            if not 2.0 ** -21 <= base < math.inf:
                raise ValueError(f"base={base} must be finite and 2^-21 or more")
            freqs = torch.tensor([float(base) ** (-i / dims) for i in range(0, dims, 2)], dtype=torch.float64, device=torch.device("cuda", torch.cuda.current_device()))
        if freqs.dim() != 1 or freqs.dtype != torch.float64 or not freqs.is_contiguous() or not 2 <= 2 * freqs.shape[0] <= head_dim:
            raise ValueError(f"freqs must be a contiguous float64 vector of 1 to {head_dim // 2}")
        if dims is not None and dims != 2 * freqs.shape[0]:
            raise ValueError(f"{freqs.shape[0]} frequencies turn {2 * freqs.shape[0]} columns, not dims={dims}")
        self.ctx, self.head_dim, self.dims, self.pairs, self.freqs = ctx, head_dim, 2 * freqs.shape[0], pairs, freqs
        self._desc, self._rows = pimdl.RotaryDesc(freqs.data_ptr(), self.dims, pimdl.PAIRS[pairs]), pimdl.RotateDesc
        self._lib = pimdl.lib()

    def _heads(self, shape, name):
        if len(shape) != 2 or shape[1] % self.head_dim:
            raise ValueError(f"{name} must be [tokens][heads * {self.head_dim}]")
        return shape[1] // self.head_dim

    def check_fits(self, cache):
        """Refuses what PagedCache.append(..., rotary=self) could not do."""
        if self.head_dim != cache.head_dim:
            raise ValueError(f"a rotation of heads of {self.head_dim} over a cache of heads of {cache.head_dim}")

    def rotate(self, q, k, q_out, k_out, starts, positions=None):
        """Turns whole sequences, which begin at position 0: q, q_out [tokens][heads * head_dim] and k, k_out [tokens][kv_heads * head_dim], packed, sequence b
        at rows starts[b] .. starts[b + 1] - 1.  An output may be its input.  `positions`: an int32 vector of the tokens' own positions instead."""
        q_shape, k_shape = q.shape, k.shape
        if q_shape != q_out.shape or k_shape != k_out.shape or q_shape[0] != k_shape[0]:
            raise ValueError("q and q_out, and k and k_out, must have one shape, all four one number of rows")
        if not q.dtype == k.dtype == q_out.dtype == k_out.dtype:
            raise ValueError("q, k, q_out and k_out must have one type")
        heads, kv_heads, tokens = self._heads(q_shape, "q"), self._heads(k_shape, "k"), q_shape[0]
        qa, qs, dtype = _packed(q, q_shape[1], "q")
        ka, ks, _ = _packed(k, k_shape[1], "k")
        qo, qos, _ = _packed(q_out, q_shape[1], "q_out")
        ko, kos, _ = _packed(k_out, k_shape[1], "k_out")
        at, n = _int_list(starts, "starts")
        if n < 1:
            raise ValueError("starts must hold one number more than there are sequences")
        pa = None
        if positions is not None:
            pa, m = _int_list(positions, "positions")
            if m != tokens:
                raise ValueError("positions must hold a number for each token")
        d = self._rows(qa, ka, qo, ko, at, pa, n - 1, tokens, heads, kv_heads, self.head_dim, qs, ks, qos, kos, dtype)
        self.ctx._check(self._lib.pimdl_rotate(self.ctx._h, self._desc, d))


class DraftTree:
    """What the nodes of the trees of a batch see of each other: masks int32 [tokens][words] (bit j of row t: node j of t's sequence is t or one of
    its ancestors) and depths int32 [tokens] (how many ancestors t has), for up to `tokens` tokens in trees of up to `most` nodes (1024)."""

    def __init__(self, ctx, pimdl, tokens, most=64):
        if tokens < 0 or not 1 <= most <= 1024:
            raise ValueError(f"tokens={tokens} and most={most}: trees have 1 to 1024 nodes")
        dev = torch.device("cuda", torch.cuda.current_device())
        masks, depths = torch.zeros(tokens, -(-most // 32), device=dev, dtype=torch.int32), torch.zeros(tokens, device=dev, dtype=torch.int32)
        # (see PagedCache: they are there when this returns)
        if not torch.cuda.is_current_stream_capturing():
            torch.cuda.current_stream(dev).synchronize()
        self._bind(ctx, pimdl, masks, depths)

    @classmethod
    def over(cls, ctx, pimdl, masks, depths):
        """Over tensors that exist already; they stay the caller's."""
        self = cls.__new__(cls)
        self._bind(ctx, pimdl, masks, depths)
        return self

    def _bind(self, ctx, pimdl, masks, depths):
        if masks.dim() != 2 or depths.shape != masks.shape[:1] or masks.dtype != torch.int32 or depths.dtype != torch.int32:
            raise ValueError("masks must be int32 [tokens][words], depths int32 [tokens]")
        if not 1 <= masks.shape[1] <= 32:
            raise ValueError(f"{masks.shape[1]} words: 1 to 32, of 32 nodes each")
        if not masks.is_contiguous() or not depths.is_contiguous() or masks.device != depths.device:
            raise ValueError("masks and depths must be contiguous and on one GPU")
        self.ctx, self.masks, self.depths = ctx, masks, depths
        self._readers = weakref.WeakSet()  # contexts that have read it and that nothing orders with its own
        self._lib, self._desc = pimdl.lib(), pimdl.TreeDesc(masks.data_ptr(), depths.data_ptr(), masks.shape[1])

    def check_tokens(self, tokens):
        """Refuses batches of more tokens than there is room for."""
        if tokens > self.masks.shape[0]:
            raise ValueError(f"{tokens} tokens: the tree has room for {self.masks.shape[0]}")

    def order(self, ctx):
        """Before calls of `ctx` that read the tree: refuses a context that runs on another stream than the tree's, where one of them was given (set_stream).  Where each has its
        own, which nobody else can order, the host waits, here for `build` and there for these calls."""
        if ctx.in_order_with(self.ctx):
            return
        if ctx.stream is not None or self.ctx.stream is not None:
            raise ValueError("the tree's context runs on another stream than the cache's: nothing orders their calls")
        if self.ctx._h:  # (not closed)
            self.ctx.synchronize()
        self._readers.add(ctx)

    def build(self, parents, starts):
        """Token t, the (t - starts[b])-th node of row b's tree, follows node parents[t] of that tree, or, with -1, what the sequence has in the cache; a parent stands before
        its children.  A tree of more nodes than there are bits is left empty: its tokens see nothing of each other, not even themselves."""
        pa, n = _int_list(parents, "parents")
        at, m = _int_list(starts, "starts")
        if m < 1:
            raise ValueError("starts must hold one number more than there are sequences")
        self.check_tokens(n)
        for ctx in self._readers:
            if ctx._h:
                ctx.synchronize()
        self._readers.clear()
        self.ctx._check(self._lib.pimdl_tree_build(self.ctx._h, pa, at, m - 1, n, self._desc.words, self._desc.masks, self._desc.depths))


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
        self._row_bytes = head_dim * k.element_size()
        self._pools = (ctypes.c_void_p * 2)(k.data_ptr(), v.data_ptr())
        self._book = pimdl.PageBook(tables.data_ptr(), lengths.data_ptr(), refs.data_ptr(), self.lacking.data_ptr(), tables.shape[0], tables.shape[1], pages,
                                    page_tokens, ctypes.cast(self._pools, ctypes.POINTER(ctypes.c_void_p)), 2, layers, layer_bytes // max(pages, 1))

    def _batch(self, starts, seqs):
        at, n = _int_list(starts, "starts")
        if n < 1:
            raise ValueError("starts must hold one number more than there are sequences")
        if seqs is None:
            return None, at, n - 1
        to, m = _int_list(seqs, "seqs")
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

    def append(self, layer, k, v, starts, seqs=None, rotary=None, q=None, q_out=None, tree=None):
        """New tokens' keys and values [tokens][kv_heads * head_dim] into the last positions of their sequences (whose room `reserve` has made).  With `rotary`
        the keys are turned by those positions on the way, and queries q [tokens][heads * head_dim], if any, into q_out (which may be q); with `tree` by the
        positions that their nodes have (the draft's first one, and the node's depth on top).  Without `rotary` a tree changes nothing here."""
        if k.shape != v.shape or k.stride() != v.stride() or k.dtype != v.dtype:
            raise ValueError("k and v must have one shape, stride and type")
        ka, ks, kt = _packed(k, self.kv_heads * self.head_dim, "k")
        to, at, batch = self._batch(starts, seqs)
        if tree is not None:
            tree.check_tokens(k.shape[0])
            tree.order(self.ctx)
        if rotary is not None:
            rotary.check_fits(self)
            depths = None if tree is None else tree._desc.depths
            if q is None and q_out is not None and q_out.numel():  # (one without columns takes none)
                raise ValueError("q_out without q: there are no queries to turn")
            heads = qa = qo = qs = qos = 0
            if q is not None:
                if q_out is None or q.shape != q_out.shape or q.dtype != k.dtype or q_out.dtype != k.dtype or q.shape[:1] != k.shape[:1]:
                    raise ValueError("q and q_out must have one shape, and k's type and number of rows")
                heads = rotary._heads(q.shape, "q")
                qa, qs, _ = _packed(q, heads * self.head_dim, "q")
                qo, qos, _ = _packed(q_out, heads * self.head_dim, "q_out")
            self.ctx._check(self._lib.pimdl_cache_append_rotary(self.ctx._h, self._of(layer), to, at, batch, k.shape[0], ka, v.data_ptr(), ks, kt, rotary._desc, depths,
                                                                qa, qo, heads, qs, qos))
            return
        if q is not None or (q_out is not None and q_out.numel()):
            raise ValueError("queries are turned by a rotary: none is given")
        self.ctx._check(self._lib.pimdl_cache_append(self.ctx._h, self._of(layer), to, at, batch, k.shape[0], ka, v.data_ptr(), ks, kt))

    def attend(self, layer, q, out, starts, heads, seqs=None, left=None, sinks=0, scale=None, tree=None):
        """Causal attention of the new tokens (q, out: [tokens][heads * head_dim]) over everything that their sequences have in the cache, or, with
        `left`, over the `left` positions before each of them and the first `sinks`.  With `tree` the new tokens of a sequence see what it had before, themselves and
        their ancestors."""
        columns = heads * self.head_dim
        if q.shape != out.shape or q.dtype != out.dtype:
            raise ValueError("q and out must have one shape and type")
        qa, qs, qt = _packed(q, columns, "q")
        oa, os_, _ = _packed(out, columns, "out")
        left = self._unlimited if left is None else left
        if not (0 <= left <= self._unlimited and 0 <= sinks <= self._unlimited):
            raise ValueError(f"left={left} and sinks={sinks} must be counts of positions, below 2^32")
        to, at, batch = self._batch(starts, seqs)
        scale = 1.0 / math.sqrt(self.head_dim) if scale is None else scale
        if tree is not None:
            tree.check_tokens(q.shape[0])
            tree.order(self.ctx)
            self.ctx._check(self._lib.pimdl_attention_tree(self.ctx._h, self._of(layer), to, at, batch, q.shape[0], tree._desc, qa, oa, heads, qs, os_, qt, left, sinks, scale))
            return
        self.ctx._check(self._lib.pimdl_attention_paged(self.ctx._h, self._of(layer), to, at, batch, q.shape[0], qa, oa, heads, qs, os_, qt, left, sinks, scale))

    def reserve(self, seqs, counts):
        """Makes sequence seqs[i] counts[i] positions longer (pages: the lowest free ones)."""
        a, n = _int_list(seqs, "seqs")
        c, m = _int_list(counts, "counts")
        if n != m:
            raise ValueError("seqs and counts must have one length")
        self.ctx._check(self._lib.pimdl_pages_reserve(self.ctx._h, self._book, a, c, n))

    def fork(self, parents, children):
        """Gives each empty sequence children[i] what parents[i] has: whole pages are shared, a partly filled last one is copied."""
        a, n = _int_list(parents, "parents")
        c, m = _int_list(children, "children")
        if n != m:
            raise ValueError("parents and children must have one length")
        self.ctx._check(self._lib.pimdl_pages_fork(self.ctx._h, self._book, a, c, n))

    def free(self, seqs):
        """Empties the sequences and gives their pages back."""
        a, n = _int_list(seqs, "seqs")
        self.ctx._check(self._lib.pimdl_pages_free(self.ctx._h, self._book, a, n))

    def accept(self, tree, last, kept, starts, seqs=None):
        """Ends the sequences behind a branch of their trees: of row b, whose nodes are the newest starts[b + 1] - starts[b] positions, the nodes from the root to last[b]
        (-1: none) move to the front of those positions, the others go, and their pages are free again.  kept[b]: how many stayed, -1 where the sequence has been
        left as it was (last[b] is no node of it; it is listed twice; the last reserve lacked pages; a fork made meanwhile holds the draft's pages too)."""
        to, at, batch = self._batch(starts, seqs)
        la, n = _int_list(last, "last")
        ka, m = _int_list(kept, "kept")
        if n != batch or m != batch:
            raise ValueError("last and kept must hold a number for each sequence of the batch")
        tree.order(self.ctx)
        self.ctx._check(self._lib.pimdl_pages_accept(self.ctx._h, self._book, to, at, batch, tree.masks.shape[0], tree._desc, la, self._row_bytes, ka))

    def compact(self):
        """Moves all pages in use to the front of the cache."""
        self.ctx._check(self._lib.pimdl_pages_compact(self.ctx._h, self._book))

    def copy(self, src, dst):
        """Copies page src[i] to page dst[i] in every layer."""
        a, n = _int_list(src, "src")
        c, m = _int_list(dst, "dst")
        if n != m:
            raise ValueError("src and dst must have one length")
        self.ctx._check(self._lib.pimdl_pages_copy(self.ctx._h, self._book, a, c, n))
