"""The operators of serving with a paged cache, as cases that can be timed: in a plain form, and as the framework's own calls.

Five kinds of pass:

  window   attention of whole sequences of a ragged, packed batch in which position p sees key j where j <= p + right and
           (j + left >= p or j < sinks): the neighbourhood of a token and the first tokens (Context.attention_window_ptr).
  paged    attention of the newest tokens of each sequence over its pages of the cache, causal, with or without a window:
           single tokens, chunks of a prompt, or both in one batch (PagedCache.attend).
  append   new keys and values, rounded to the cache's type and written into the pages (PagedCache.append).
  beams    one step of a beam search: the chosen beams are forked into free sequences, the old ones freed (PagedCache.fork, free).
  compact  the live pages of a cache that has holes move to its front (PagedCache.compact).

`own` says which form `run` computes.  Lengths are spread over their range by the golden ratio, so that a batch is as ragged as
its range and the work of a case does not depend on the seed.  Activations are N(0, 1), as layer normalisation leaves them; the
cache's pages hold such rows too, pages and parts of pages that no sequence holds among them.
"""
import math
import os
import sys

import torch

own = False

_DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
_BYTES = {"f32": 4, "f16": 2, "bf16": 2}
_package = _context = _pages = None


# ------------------------------------------------------------------------------------------------ the cases

def _window(batch, low, high, heads, kv_heads, head_dim, left, right, sinks, dtype):
    return {"kind": "window", "batch": batch, "low": low, "high": high, "heads": heads, "kv_heads": kv_heads, "head_dim": head_dim,
            "left": left, "right": right, "sinks": sinks, "dtype": dtype}


def _paged(batch, new_low, new_high, low, high, heads, kv_heads, head_dim, page_tokens, dtype, cache, left=-1, sinks=0):
    return {"kind": "paged", "batch": batch, "new_low": new_low, "new_high": new_high, "low": low, "high": high, "heads": heads,
            "kv_heads": kv_heads, "head_dim": head_dim, "page_tokens": page_tokens, "dtype": dtype, "cache": cache, "left": left, "sinks": sinks}


def _append(batch, new_low, new_high, low, high, kv_heads, head_dim, page_tokens, dtype, cache):
    return {"kind": "append", "batch": batch, "new_low": new_low, "new_high": new_high, "low": low, "high": high, "kv_heads": kv_heads,
            "head_dim": head_dim, "page_tokens": page_tokens, "dtype": dtype, "cache": cache}


def _beams(prompts, beams, low, high, layers, kv_heads, head_dim, page_tokens, cache):
    return {"kind": "beams", "prompts": prompts, "beams": beams, "low": low, "high": high, "layers": layers, "kv_heads": kv_heads,
            "head_dim": head_dim, "page_tokens": page_tokens, "cache": cache}


def _compact(pages, live, seqs, layers, kv_heads, head_dim, page_tokens, cache):
    return {"kind": "compact", "pages": pages, "live": live, "seqs": seqs, "layers": layers, "kv_heads": kv_heads, "head_dim": head_dim,
            "page_tokens": page_tokens, "cache": cache}


def listed():
    return [
        # one short text through a layer of BERT-base's heads: launches and latency
        {"name": "window_one_text_f32", **_window(1, 128, 128, 12, 12, 64, 32, 32, 1, "f32")},
        # long documents through the same layer: 256 neighbours on both sides and the first token, which stands for the document
        {"name": "window_documents_f32", **_window(6, 1000, 4096, 12, 12, 64, 256, 256, 1, "f32")},
        # prompts with shared key heads, causal, a window of 1024 and four first tokens that stay
        {"name": "window_prompts_bf16", **_window(6, 1500, 4096, 32, 8, 128, 1023, 0, 4, "bf16")},
        # one sequence of the 12-head layer a token at a time: fp32 activations over a cache in halves
        {"name": "decode_one_f32_over_f16", **_paged(1, 1, 1, 777, 777, 12, 12, 64, 16, "f32", "f16")},
        # a serving batch, each sequence at a length of its own
        {"name": "decode_batch_bf16", **_paged(64, 1, 1, 1, 8191, 32, 8, 128, 32, "bf16", "bf16")},
        # two very long contexts: few rows, and the work is along the keys
        {"name": "decode_long_f16", **_paged(2, 1, 1, 98765, 131071, 16, 2, 128, 64, "f16", "f16")},
        # chunks of prompts in the framework's own type over a cache of it; 16 heads of 80, as the large vision transformer has
        {"name": "chunk_f32", **_paged(3, 300, 512, 500, 3000, 16, 16, 80, 16, "f32", "f32")},
        # a mixed batch: some sequences take a chunk of their prompt, some a token; window of 4096 with four first tokens
        {"name": "chunk_mixed_bf16", **_paged(16, 1, 512, 100, 6000, 32, 8, 128, 16, "bf16", "bf16", 4095, 4)},
        # one new token for each of 64 sequences into a cache in halves
        {"name": "append_tokens_f32_to_f16", **_append(64, 1, 1, 0, 2000, 12, 64, 16, "f32", "f16")},
        # whole prompts into the cache
        {"name": "append_prompts_bf16", **_append(12, 500, 4096, 0, 500, 8, 128, 32, "bf16", "bf16")},
        # a beam search's step in a model of 12 layers: only the partly filled last pages are copied
        {"name": "beams_f16", **_beams(8, 4, 200, 2000, 12, 12, 64, 16, "f16")},
        # a cache of 12 layers, a third of whose pages have been freed here and there
        {"name": "compact_bf16", **_compact(4096, 0.66, 48, 12, 8, 128, 16, "bf16")},
    ]


def draw(rng):
    def spread(a, b):
        return min(b, max(a, round(math.exp(rng.uniform(math.log(a), math.log(b + 1))))))

    def heads():
        kv = rng.choice([1, 2, 3, 4, 8, 12])
        return kv * rng.choice([1, 1, 2, 3, 4, 8]), kv, rng.choice([32, 64, 64, 80, 96, 128, 128])

    kind = rng.choice(["window", "window", "paged", "paged", "paged", "paged", "append", "beams", "compact"])
    dtype = rng.choice(["f32", "f16", "bf16"])
    cache = rng.choice(["f32", "f16", "bf16"]) if dtype == "f32" else dtype
    page_tokens = rng.choice([16, 32, 64, 128])
    while True:
        if kind == "window":
            h, kv, hd = heads()
            high = spread(16, 4096)
            c = _window(spread(1, 32), spread(1, high), high, h, kv, hd, spread(1, 2048), rng.choice([0, 0, spread(1, 512)]), rng.choice([0, 1, 4, spread(1, 64)]), dtype)
        elif kind == "paged":
            h, kv, hd = heads()
            decode, high = rng.random() < 0.5, spread(16, 65536)
            new = 1 if decode else spread(2, 700)
            c = _paged(spread(1, 128), 1 if decode else spread(1, new), new, spread(1, high), high, h, kv, hd, page_tokens, dtype, cache,
                       rng.choice([-1, -1, spread(1, 8192)]), rng.choice([0, 4]))
        elif kind == "append":
            h, kv, hd = heads()
            new, high = spread(1, 4096), spread(1, 4096)
            c = _append(spread(1, 128), spread(1, new), new, spread(1, high), high, kv, hd, page_tokens, dtype, cache)
        elif kind == "beams":
            h, kv, hd = heads()
            high = spread(10, 2000)
            c = _beams(spread(1, 16), rng.choice([2, 3, 4, 8]), spread(1, high), high, rng.choice([1, 2, 6, 12]), kv, hd, page_tokens, cache)
        else:
            h, kv, hd = heads()
            pages = spread(64, 4096)
            c = _compact(pages, round(rng.uniform(0.3, 0.9), 2), spread(1, min(64, pages // 8)), rng.choice([1, 2, 6, 12]), kv, hd, page_tokens, cache)
        if _fits(c):
            return c


def _fits(c):
    """No more than the largest listed cases: by what the plain form has to hold, by operations and by bytes."""
    w = work(c)
    if c["kind"] in ("window", "paged"):
        long = c["high"] if c["kind"] == "window" else c["high"] + c["new_high"]
        new = c["high"] if c["kind"] == "window" else c["new_high"]
        if c["batch"] * c["heads"] * new * long > 6 * 32 * 4096 * 4096 // 4 or c["batch"] * c["kv_heads"] * long * c["head_dim"] > 64 * 8 * 8192 * 128:
            return False
        return w["flops"] <= 3e11 and w["bytes"] <= 1.2e9
    if c["kind"] in ("beams", "compact"):
        count = c["pages"] if c["kind"] == "compact" else (c["prompts"] * -(-c["high"] // c["page_tokens"]) + 2 * c["prompts"] * c["beams"])
        if count * _page_bytes(c) > 4e9:
            return False
    return w["bytes"] <= 2.5e9


def _spread(count, low, high):
    return [low + int((high - low + 1) * ((0.618033988749895 * (i + 1)) % 1.0)) for i in range(count)]


def _new_counts(c):
    n = _spread(c["batch"], c["new_low"], c["new_high"])
    if c["new_high"] > 1 and c["new_low"] == 1:  # a mixed batch: every other sequence takes a single token
        n = [1 if i % 2 else x for i, x in enumerate(n)]
    return n


def _page_bytes(c):
    return 2 * c["layers"] * c["kv_heads"] * c["page_tokens"] * c["head_dim"] * _BYTES[c["cache"]]


def _seen(p, length, left, right, sinks):
    """How many keys the query at position p sees."""
    last = min(length - 1, p + right)
    first = max(0, p - left) if left >= 0 else 0
    return max(0, last - first + 1) + max(0, min(sinks, first, last + 1))


def work(case):
    c = case
    if c["kind"] == "window":
        lens, e = _spread(c["batch"], c["low"], c["high"]), _BYTES[c["dtype"]]
        pairs = sum(_seen(p, n, c["left"], c["right"], c["sinks"]) for n in lens for p in range(n))
        return {"bytes": sum(lens) * c["head_dim"] * (2 * c["heads"] + 2 * c["kv_heads"]) * e + 4 * (c["batch"] + 1), "flops": 4 * c["head_dim"] * c["heads"] * pairs}
    if c["kind"] == "paged":
        new, old = _new_counts(c), _spread(c["batch"], c["low"], c["high"])
        pairs = rows = 0
        for n, o in zip(new, old):
            pairs += sum(_seen(o + i, o + n, c["left"], 0, c["sinks"]) for i in range(n))
            first = max(0, o - c["left"]) if c["left"] >= 0 else 0
            rows += o + n - first + min(c["sinks"], first)
        kv = 2 * rows * c["kv_heads"] * c["head_dim"] * _BYTES[c["cache"]]
        return {"bytes": kv + 2 * sum(new) * c["heads"] * c["head_dim"] * _BYTES[c["dtype"]] + 4 * rows // c["page_tokens"], "flops": 4 * c["head_dim"] * c["heads"] * pairs}
    if c["kind"] == "append":
        return {"bytes": 2 * sum(_new_counts(c)) * c["kv_heads"] * c["head_dim"] * (_BYTES[c["dtype"]] + _BYTES[c["cache"]]), "flops": 0}
    if c["kind"] == "beams":
        lens = _spread(c["prompts"], c["low"], c["high"])
        filled = sum(n % c["page_tokens"] for n in lens) * c["beams"]  # rows of the partly filled pages, read and written
        rows = sum(-(-n // c["page_tokens"]) for n in lens) * c["beams"]  # entries of the tables: read, written for the children, cleared for the parents
        return {"bytes": 2 * filled * _page_bytes(c) // c["page_tokens"] + 4 * 3 * rows, "flops": 0}
    live, pages = _live(c)
    moved = sum(1 for p in live if p >= len(live))
    return {"bytes": 2 * moved * _page_bytes(c) + 4 * (2 * pages + 2 * len(live)), "flops": 0}


def _live(c):
    """The pages that a fragmented cache holds: spread over all of it."""
    pages, want = c["pages"], max(1, int(c["pages"] * c["live"]))
    order = sorted(range(pages), key=lambda p: (0.618033988749895 * (p + 1)) % 1.0)
    return sorted(order[:want]), pages


# ------------------------------------------------------------------------------------------------ what a program has in hand

def _rand(gen, *shape, dtype=torch.float32):
    return torch.randn(shape, device="cuda", generator=gen, dtype=torch.float32 if dtype == torch.float32 else torch.float16).to(dtype)


def _starts(counts):
    at = [0]
    for n in counts:
        at.append(at[-1] + n)
    return torch.tensor(at, dtype=torch.int32, device="cuda")


def _tables(gen, lens, page_tokens, pages, width):
    """Each sequence's pages, anywhere in the cache."""
    order, at, rows = torch.randperm(pages, generator=gen, device="cuda").tolist(), 0, []
    for n in lens:
        k = -(-n // page_tokens)
        rows.append(order[at:at + k] + [-1] * (width - k))
        at += k
    return torch.tensor(rows, dtype=torch.int32, device="cuda")


def prepare(case, seed):
    c = case
    gen = torch.Generator(device="cuda").manual_seed(seed)
    if c["kind"] == "window":
        lens, dt = _spread(c["batch"], c["low"], c["high"]), _DTYPES[c["dtype"]]
        n, d, kd = sum(lens), c["heads"] * c["head_dim"], c["kv_heads"] * c["head_dim"]
        return {**c, "qkv": _rand(gen, n, d + 2 * kd, dtype=dt), "out": torch.zeros(n, d, device="cuda", dtype=dt), "starts": _starts(lens),
                "max_new": max(lens), "max_len": max(lens)}
    if c["kind"] in ("paged", "append"):
        new, old = _new_counts(c), _spread(c["batch"], c["low"], c["high"])
        lens, dt, ct, pt = [a + b for a, b in zip(new, old)], _DTYPES[c["dtype"]], _DTYPES[c["cache"]], c["page_tokens"]
        need = sum(-(-x // pt) for x in lens)
        pages, width = need + need // 8 + 1, -(-max(lens) // pt)
        s = {**c, "starts": _starts(new), "lengths": torch.tensor(lens, dtype=torch.int32, device="cuda"),
             "tables": _tables(gen, lens, pt, pages, width), "refs": torch.zeros(pages, dtype=torch.int32, device="cuda"), "max_new": max(new), "max_len": max(lens)}
        s["refs"][s["tables"][s["tables"] >= 0].long()] = 1
        for name in ("k_pages", "v_pages"):
            s[name] = _rand(gen, 1, pages, c["kv_heads"], pt, c["head_dim"], dtype=ct)
        if c["kind"] == "paged":
            s["q"] = _rand(gen, sum(new), c["heads"] * c["head_dim"], dtype=dt)
            s["out"] = torch.zeros(sum(new), c["heads"] * c["head_dim"], device="cuda", dtype=dt)
        else:
            s["k"], s["v"] = (_rand(gen, sum(new), c["kv_heads"] * c["head_dim"], dtype=dt) for _ in range(2))
        return s
    pt, ct = c["page_tokens"], _DTYPES[c["cache"]]
    if c["kind"] == "beams":
        per, lens = c["beams"], _spread(c["prompts"], c["low"], c["high"])
        seqs, width = 2 * c["prompts"] * per, -(-max(lens) // pt) + 1
        rows = [[-1] * width for _ in range(seqs)]
        lengths, at = [0] * seqs, 0
        for i, n in enumerate(lens):  # the whole pages of a prompt are shared by its beams, each beam has a last page of its own
            whole = list(range(at, at + n // pt))
            at += n // pt
            for b in range(per):
                rows[i * per + b][:len(whole)] = whole
                lengths[i * per + b] = n
                if n % pt:
                    rows[i * per + b][len(whole)] = at
                    at += 1
        pages = at + c["prompts"] * per + 1
        first = torch.arange(c["prompts"] * per, dtype=torch.int32, device="cuda")
        chosen = torch.randint(0, per, (c["prompts"] * per,), generator=gen, device="cuda", dtype=torch.int32) + first // per * per
        half = c["prompts"] * per
        s = {**c, "turn": 0, "chosen": (chosen, chosen + half), "olds": (first, first + half), "tables": torch.tensor(rows, dtype=torch.int32, device="cuda"),
             "lengths": torch.tensor(lengths, dtype=torch.int32, device="cuda")}
        held = s["tables"][s["tables"] >= 0].long()
        s["refs"] = torch.zeros(pages, dtype=torch.int32, device="cuda").index_add_(0, held, torch.ones_like(held, dtype=torch.int32))
    else:
        live, pages = _live(c)
        order = [live[i] for i in torch.randperm(len(live), generator=gen, device="cuda").tolist()]
        seqs, width = c["seqs"], -(-len(live) // c["seqs"])
        rows = [order[i * width:(i + 1) * width] for i in range(seqs)]
        s = {**c, "tables": torch.tensor([r + [-1] * (width - len(r)) for r in rows], dtype=torch.int32, device="cuda"),
             "lengths": torch.tensor([len(r) * pt for r in rows], dtype=torch.int32, device="cuda"), "refs": torch.zeros(pages, dtype=torch.int32, device="cuda")}
        s["refs"][s["tables"][s["tables"] >= 0].long()] = 1
        s["broken_tables"], s["broken_refs"] = s["tables"].clone(), s["refs"].clone()
    for name in ("k_pages", "v_pages"):
        s[name] = _rand(gen, c["layers"], pages, c["kv_heads"], pt, c["head_dim"], dtype=ct)
    return s


# ------------------------------------------------------------------------------------------------ one pass

def _ctx():
    """One context for the process, on torch's stream, as a serving program holds it."""
    global _package, _context, _pages
    if _context is None:
        root = os.getcwd()
        if root not in sys.path:
            sys.path.insert(0, root)
        from __graft_entry__ import load_package
        _package = load_package()
        from pim_dl_asplos_amd import kvcache as _pages
        _context = _package.Context(torch.cuda.current_device())
        _context.set_stream(torch.cuda.current_stream().cuda_stream)
    return _context


def _cache(s):
    """The program's handle of its cache."""
    if "handle" not in s:
        ctx = _ctx()
        s["handle"] = _pages.PagedCache.over(ctx, _package, s["k_pages"], s["v_pages"], s["tables"], s["lengths"], s["refs"])
    return s["handle"]


def run(state):
    return {"window": _run_window, "paged": _run_paged, "append": _run_append, "beams": _run_beams, "compact": _run_compact}[state["kind"]](state)


def _run_window(s):
    h, kv, hd = s["heads"], s["kv_heads"], s["head_dim"]
    d, kd, qkv, out = h * hd, kv * hd, s["qkv"], s["out"]
    if own:
        ctx, e, at = _ctx(), qkv.element_size(), qkv.data_ptr()
        ctx.attention_window_ptr(at, at + d * e, at + (d + kd) * e, out.data_ptr(), s["starts"].data_ptr(), s["batch"], out.shape[0], h, kv, hd,
                                 d + 2 * kd, d + 2 * kd, d, s["left"], s["right"], s["sinks"], 1 / math.sqrt(hd), _package.DTYPES[s["dtype"]])
        return out
    rows, here = _rows(s["starts"], s["max_new"])
    parts = qkv[rows].float()  # [batch][max_new][...]
    q, k, v = parts[..., :d].unflatten(-1, (h, hd)), parts[..., d:d + kd].unflatten(-1, (kv, hd)), parts[..., d + kd:].unflatten(-1, (kv, hd))
    p = torch.arange(s["max_new"], device=qkv.device)
    near = (p[None, :] <= p[:, None] + s["right"]) & ((p[None, :] + s["left"] >= p[:, None]) | (p[None, :] < s["sinks"]))
    o = _attention(q, k, v, near[None] & here[:, None, :], 1 / math.sqrt(hd))
    out[rows[here]] = o[here].flatten(1).to(out.dtype)
    return out


def _rows(starts, most):
    """Rows of the packed tokens as [batch][most], and which of them exist."""
    at = torch.arange(most, device=starts.device)
    here = at[None, :] < (starts[1:] - starts[:-1])[:, None]
    return torch.where(here, starts[:-1, None] + at, 0).long(), here


def _attention(q, k, v, seen, scale):
    """q [batch][new][heads][hd], k and v [batch][keys][kv_heads][hd], seen [batch][new][keys]: zeros where nothing is seen."""
    b, n, h, hd = q.shape
    kv = k.shape[2]
    qh = q.reshape(b, n, kv, h // kv, hd).permute(0, 2, 3, 1, 4).reshape(b * kv, h // kv * n, hd)
    kh, vh = (x.permute(0, 2, 1, 3).reshape(b * kv, -1, hd) for x in (k, v))
    s = torch.bmm(qh, kh.transpose(1, 2).contiguous()).mul_(scale).reshape(b, kv, h // kv, n, -1)
    s.masked_fill_(~seen[:, None, None], -math.inf)
    most = s.amax(-1, keepdim=True)
    s = s.sub_(torch.where(most == -math.inf, 0.0, most)).exp_()
    total = s.sum(-1, keepdim=True)
    o = torch.bmm(s.reshape(b * kv, h // kv * n, -1), vh).reshape(b, kv, h // kv, n, hd) / torch.where(total > 0, total, 1.0)
    return o.permute(0, 3, 1, 2, 4).reshape(b, n, h, hd)


def _run_paged(s):
    h, kv, hd, out = s["heads"], s["kv_heads"], s["head_dim"], s["out"]
    if own:
        _cache(s).attend(0, s["q"], out, s["starts"], h, left=s["left"] if s["left"] >= 0 else None, sinks=s["sinks"])
        return out
    pt, starts, lengths = s["page_tokens"], s["starts"], s["lengths"]
    rows, here = _rows(starts, s["max_new"])
    key = torch.arange(s["tables"].shape[1] * pt, device=out.device)
    held = key[None, :] < lengths[:, None]
    pages = s["tables"].clamp(min=0).long()
    k, v = (x[0][pages].float().permute(0, 1, 3, 2, 4).reshape(s["batch"], -1, kv, hd) for x in (s["k_pages"], s["v_pages"]))
    v = torch.where(held[:, :, None, None], v, 0.0)
    place = lengths[:, None] - (starts[1:] - starts[:-1])[:, None] + torch.arange(s["max_new"], device=out.device)
    seen = (key[None, None, :] <= place[:, :, None]) & held[:, None, :]
    if s["left"] >= 0:
        seen &= (key[None, None, :] + s["left"] >= place[:, :, None]) | (key < s["sinks"])[None, None, :]
    o = _attention(s["q"][rows].float().unflatten(-1, (h, hd)), k, v, seen, 1 / math.sqrt(hd))
    out[rows[here]] = o[here].flatten(1).to(out.dtype)
    return out


def _run_append(s):
    if own:
        _cache(s).append(0, s["k"], s["v"], s["starts"])
        return s["k_pages"], s["v_pages"]
    pt, starts, n = s["page_tokens"], s["starts"].long(), s["k"].shape[0]
    seq = torch.searchsorted(starts[1:].contiguous(), torch.arange(n, device=starts.device), right=True)
    place = s["lengths"].long()[seq] - starts[seq + 1] + torch.arange(n, device=starts.device)
    page = s["tables"].long()[seq, place // pt]
    for pool, x in ((s["k_pages"], s["k"]), (s["v_pages"], s["v"])):
        pool[0][page, :, place % pt] = x.unflatten(-1, (s["kv_heads"], s["head_dim"])).to(pool.dtype)
    return s["k_pages"], s["v_pages"]


def _run_beams(s):
    turn, s["turn"] = s["turn"], 1 - s["turn"]
    parents, children, old = s["chosen"][turn], s["olds"][1 - turn], s["olds"][turn]
    tables, lengths, refs = s["tables"], s["lengths"], s["refs"]
    if own:
        cache = _cache(s)
        cache.fork(parents, children)
        cache.free(old)
        return s["k_pages"], s["v_pages"], tables, lengths, refs
    pt, count = s["page_tokens"], lengths[parents.long()].long()
    rows = tables[parents.long()]
    whole = torch.arange(rows.shape[1], device=rows.device)[None, :] < (count // pt)[:, None]
    refs.index_add_(0, rows[whole].long(), torch.ones_like(rows[whole]))
    part = torch.nonzero(count % pt).flatten()
    fresh = torch.nonzero(refs == 0).flatten()[:part.numel()]
    src = rows[part, count[part] // pt].long()
    for pool in (s["k_pages"], s["v_pages"]):
        pool[:, fresh] = pool[:, src]
    rows[part, count[part] // pt] = fresh.int()
    refs[fresh] = 1
    tables[children.long()], lengths[children.long()] = rows, count.int()
    gone = tables[old.long()]
    refs.index_add_(0, gone[gone >= 0].long(), -torch.ones_like(gone[gone >= 0]))
    tables[old.long()], lengths[old.long()] = -1, 0
    return s["k_pages"], s["v_pages"], tables, lengths, refs


def _run_compact(s):
    tables, refs = s["tables"], s["refs"]
    tables.copy_(s["broken_tables"])  # (as other sequences came and went)
    refs.copy_(s["broken_refs"])
    if own:
        _cache(s).compact()
        return s["k_pages"], s["v_pages"], tables, refs
    live = refs > 0
    count = int(live.sum())
    holes, movers = torch.nonzero(~live[:count]).flatten(), torch.nonzero(live[count:]).flatten() + count
    place = torch.arange(refs.numel(), device=refs.device, dtype=torch.int32)
    place[movers] = holes.int()
    for pool in (s["k_pages"], s["v_pages"]):
        pool[:, holes] = pool[:, movers]
    tables.copy_(torch.where(tables >= 0, place[tables.clamp(min=0).long()], -1))
    refs[holes] = refs[movers]
    refs[movers] = 0
    return s["k_pages"], s["v_pages"], tables, refs


# ------------------------------------------------------------------------------------------------ the definition in 64 bits

def exact(case, seed):
    s = prepare(case, seed)
    if s["kind"] in ("window", "paged"):
        return _exact_attention(s)
    if s["kind"] == "append":
        pools, at = [s["k_pages"].double(), s["v_pages"].double()], s["starts"].tolist()
        for b, n in enumerate(s["lengths"].tolist()):
            place = torch.arange(n - (at[b + 1] - at[b]), n, device="cuda")
            page = s["tables"][b].long()[place // s["page_tokens"]]
            for pool, x in zip(pools, (s["k"], s["v"])):
                pool[0, page, :, place % s["page_tokens"]] = x[at[b]:at[b + 1]].double().reshape(-1, s["kv_heads"], s["head_dim"])
        return tuple(pools)
    return None  # pages are moved as they are


def _exact_attention(s):
    """Sequence by sequence, head by head and 1024 queries at a time: softmax(q k^T / sqrt(hd)) v over the keys that each query sees."""
    h, kv, hd, at = s["heads"], s["kv_heads"], s["head_dim"], s["starts"].tolist()
    out = torch.zeros(at[-1], h, hd, device="cuda", dtype=torch.float64)
    for b in range(s["batch"]):
        n = at[b + 1] - at[b]
        if s["kind"] == "window":
            x = s["qkv"][at[b]:at[b + 1]].double()
            q, k, v = x[:, :h * hd].reshape(n, h, hd), x[:, h * hd:(h + kv) * hd].reshape(n, kv, hd), x[:, (h + kv) * hd:].reshape(n, kv, hd)
            length, left, right = n, s["left"], s["right"]
        else:
            length, left, right = int(s["lengths"][b]), s["left"] if s["left"] >= 0 else 1 << 40, 0
            page = s["tables"][b, :-(-length // s["page_tokens"])].long()
            k, v = (x[0, page].double().transpose(1, 2).reshape(-1, kv, hd)[:length] for x in (s["k_pages"], s["v_pages"]))
            q = s["q"][at[b]:at[b + 1]].double().reshape(n, h, hd)
        keys = torch.arange(length, device="cuda")
        for i in range(0, n, 1024):
            p = torch.arange(length - n + i, length - n + min(n, i + 1024), device="cuda")[:, None]
            lo = 0 if s["sinks"] or left >= length else max(0, int(p[0]) - left)
            hi = min(length, int(p[-1]) + right + 1)
            j = keys[None, lo:hi]
            hidden = (j > p + right) | ((j + left < p) & (j >= s["sinks"]))
            for a in range(kv):
                rows = q[i:i + 1024, a * (h // kv):(a + 1) * (h // kv)].transpose(0, 1).reshape(-1, hd)
                score = (rows @ k[lo:hi, a].t().contiguous()).reshape(h // kv, -1, hi - lo) / math.sqrt(hd)
                share = torch.softmax(score.masked_fill(hidden[None], -math.inf), -1)
                out[at[b] + i:at[b] + i + p.shape[0], a * (h // kv):(a + 1) * (h // kv)] = (share.reshape(-1, hi - lo) @ v[lo:hi, a].contiguous()).reshape(h // kv, -1, hd).transpose(0, 1)
    return out.reshape(at[-1], h * hd)
