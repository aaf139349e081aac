"""The operators of serving a model with rotated positions and drafted tokens, as cases that can be timed: in a plain form, and as the framework's own calls.

Five kinds of pass:

  rotate   queries and keys of whole sequences, packed, turned by their positions: the pair (a, b) of columns that belongs to frequency f becomes
           (a cos pf - b sin pf, a sin pf + b cos pf) at position p (Rotary.rotate).
  append   the newest tokens' keys, turned, and values into the pages of the cache, their queries turned (PagedCache.append with a Rotary).
  tree     what the nodes of trees of drafted tokens see of each other, as bits, and their depths, from their parents (DraftTree.build).
  verify   attention of the drafted tokens of each sequence over its pages: what was there before, itself and its ancestors, with or
           without a window (PagedCache.attend with a DraftTree).
  accept   the chosen branch of each tree moves to the front of the drafted positions, in every layer, and the sequence ends behind it
           (PagedCache.accept).

`own` says which form `run` computes.  Lengths are spread over their range by the golden ratio and trees grow by rule, so that a batch is as ragged as
its range and the work of a case does not depend on the seed.  Activations are N(0, 1), as layer normalisation leaves them; the cache's
pages hold such rows too, pages and parts of pages that no sequence holds among them.
"""
import math
import os
import sys

import torch

own = False

_DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
_BYTES = {"f32": 4, "f16": 2, "bf16": 2}
_GOLDEN = 0.618033988749895
_package = _context = _pages = None


# ------------------------------------------------------------------------------------------------ the cases

def _rotate(batch, low, high, heads, kv_heads, head_dim, dims, pairs, base, dtype):
    return {"kind": "rotate", "batch": batch, "low": low, "high": high, "heads": heads, "kv_heads": kv_heads, "head_dim": head_dim, "dims": dims,
            "pairs": pairs, "base": base, "dtype": dtype}


def _append(batch, new_low, new_high, low, high, heads, kv_heads, head_dim, dims, pairs, base, page_tokens, dtype, cache, width=-1):
    """width: of the trees that the new tokens are (see _parents); -1: they follow each other"""
    return {"kind": "append", "batch": batch, "new_low": new_low, "new_high": new_high, "low": low, "high": high, "heads": heads, "kv_heads": kv_heads,
            "head_dim": head_dim, "dims": dims, "pairs": pairs, "base": base, "page_tokens": page_tokens, "dtype": dtype, "cache": cache, "width": width}


def _tree(batch, new_low, new_high, width):
    return {"kind": "tree", "batch": batch, "new_low": new_low, "new_high": new_high, "width": width}


def _verify(batch, new_low, new_high, low, high, heads, kv_heads, head_dim, page_tokens, dtype, cache, width, left=-1, sinks=0):
    return {"kind": "verify", "batch": batch, "new_low": new_low, "new_high": new_high, "low": low, "high": high, "heads": heads, "kv_heads": kv_heads,
            "head_dim": head_dim, "page_tokens": page_tokens, "dtype": dtype, "cache": cache, "width": width, "left": left, "sinks": sinks}


def _accept(batch, new_low, new_high, low, high, layers, kv_heads, head_dim, page_tokens, cache, width):
    return {"kind": "accept", "batch": batch, "new_low": new_low, "new_high": new_high, "low": low, "high": high, "layers": layers, "kv_heads": kv_heads,
            "head_dim": head_dim, "page_tokens": page_tokens, "cache": cache, "width": width}


def listed():
    return [
        # one short text through a layer of BERT-base's heads, pairs of neighbouring columns: launches and latency
        {"name": "rotate_text_f32", **_rotate(1, 128, 128, 12, 12, 64, 64, "neighbours", 10000.0, "f32")},
        # whole prompts of a model with shared key heads, before attention without a cache
        {"name": "rotate_prompts_bf16", **_rotate(6, 1500, 4096, 32, 8, 128, 128, "halves", 10000.0, "bf16")},
        # a serving batch, one new token each: a quarter of each head's columns turned, a cache in halves
        {"name": "append_tokens_f32_to_f16", **_append(64, 1, 1, 0, 2000, 12, 12, 64, 16, "halves", 10000.0, 16, "f32", "f16")},
        # prompts into the cache, the frequencies of a model for long contexts
        {"name": "append_prompts_bf16", **_append(12, 500, 4096, 0, 500, 32, 8, 128, 128, "halves", 500000.0, 32, "bf16", "bf16")},
        # one sequence's draft: 16 nodes
        {"name": "tree_one", **_tree(1, 16, 16, 0)},
        # a batch of large drafts
        {"name": "tree_batch", **_tree(64, 100, 512, 0)},
        # one sequence of the 12-head layer with a small draft, four candidates deep and wide: fp32 over a cache in halves
        {"name": "verify_one_f32_over_f16", **_verify(1, 24, 24, 777, 777, 12, 12, 64, 16, "f32", "f16", 4)},
        # a serving batch, each sequence at a length of its own with a draft of its own
        {"name": "verify_batch_bf16", **_verify(32, 16, 64, 1, 8191, 32, 8, 128, 32, "bf16", "bf16", 0)},
        # two very long contexts: the work is along the keys
        {"name": "verify_long_f16", **_verify(2, 33, 48, 98765, 131071, 16, 2, 128, 64, "f16", "f16", 8)},
        # large drafts in the framework's own type; heads of 80, a window of 1024 with four first tokens
        {"name": "verify_window_f32", **_verify(4, 100, 250, 500, 3000, 16, 16, 80, 16, "f32", "f32", 0, 1023, 4)},
        # one sequence accepts a branch of its draft in 12 layers
        {"name": "accept_one_f16", **_accept(1, 24, 24, 777, 777, 12, 12, 64, 16, "f16", 4)},
        # a serving batch does
        {"name": "accept_batch_bf16", **_accept(64, 32, 256, 100, 2000, 12, 8, 128, 32, "bf16", 3)},
    ]


def draw(rng):
    def spread(a, b):
        return min(b, max(a, round(math.exp(rng.uniform(math.log(a), math.log(b + 1))))))

    def heads():
        kv = rng.choice([1, 2, 3, 4, 8, 12])
        return kv * rng.choice([1, 1, 2, 3, 4, 8]), kv, rng.choice([32, 64, 64, 80, 96, 128, 128])

    kind = rng.choice(["rotate", "append", "append", "tree", "verify", "verify", "verify", "verify", "accept"])
    dtype = rng.choice(["f32", "f16", "bf16"])
    cache = rng.choice(["f32", "f16", "bf16"]) if dtype == "f32" else dtype
    page_tokens = rng.choice([16, 32, 64, 128])
    width = rng.choice([0, 0, 1, spread(1, 32)])
    pairs, base = rng.choice(["halves", "neighbours"]), rng.choice([10000.0, 500000.0, 1000000.0])
    while True:
        h, kv, hd = heads()
        dims = rng.choice([hd, hd, hd // 2, 2 * rng.randint(1, hd // 2)])
        if kind == "rotate":
            high = spread(1, 4096)
            c = _rotate(spread(1, 64), spread(1, high), high, h, kv, hd, dims, pairs, base, dtype)
        elif kind == "append":
            draft = rng.random() < 0.3
            new, high = spread(1, 300 if draft else 4096), spread(1, 65536)
            c = _append(spread(1, 128), spread(1, new), new, spread(1, high), high, h, kv, hd, dims, pairs, base, page_tokens, dtype, cache, width if draft else -1)
        elif kind == "tree":
            new = spread(1, 1024)
            c = _tree(spread(1, 128), spread(1, new), new, width)
        elif kind == "verify":
            new, high = spread(1, 500), spread(16, 65536)
            c = _verify(spread(1, 128), spread(1, new), new, spread(1, high), high, h, kv, hd, page_tokens, dtype, cache, width,
                        rng.choice([-1, -1, spread(1, 8192)]), rng.choice([0, 4]))
        else:
            new, high = spread(1, 500), spread(1, 2000)
            c = _accept(spread(1, 128), spread(1, new), new, spread(1, high), high, rng.choice([1, 2, 6, 12]), kv, hd, page_tokens, cache, width)
        if _fits(c):
            return c


def _fits(c):
    """No more than the largest listed cases: by what the plain form has to hold, by operations and by bytes."""
    w = work(c)
    if c["kind"] in ("append", "verify", "accept"):
        long = c["high"] + c["new_high"]
        if c["batch"] * c["kv_heads"] * (long + c["page_tokens"]) * c["head_dim"] * c.get("layers", 1) > 32 * 8 * 8192 * 128:
            return False
        if c["kind"] == "verify" and c["batch"] * c["heads"] * c["new_high"] * long > 32 * 32 * 64 * 8192:
            return False
    if c["kind"] == "tree" and c["batch"] * (-(-c["new_high"] // 32) * 32) ** 2 > 64 * 512 * 512:
        return False
    return w["bytes"] <= (7e8 if c["kind"] in ("rotate", "append") else 6e8) and w["flops"] <= 8e10


def _spread(count, low, high):
    return [low + int((high - low + 1) * ((_GOLDEN * (i + 1)) % 1.0)) for i in range(count)]


def _parents(n, width):
    """The parents of a tree of n nodes.  width > 0: `width` candidates after the first token, each a chain, level by level (1: one chain); 0: each node hangs on any
    of those before it or on what is in the cache."""
    if width:
        return [-1 if i == 0 else 0 if i <= width else i - width for i in range(n)]
    return [int((i + 1) * ((_GOLDEN * (i + 1)) % 1.0)) - 1 for i in range(n)]


def _depths(parents):
    d = []
    for p in parents:
        d.append(0 if p < 0 else d[p] + 1)
    return d


def _last(c):
    """The node that each sequence accepts up to; -1: none"""
    new = _spread(c["batch"], c["new_low"], c["new_high"])
    return [int((n + 1) * ((_GOLDEN * (7 * b + 1)) % 1.0)) - 1 for b, n in enumerate(new)]


def _path(parents, last):
    path = []
    while last >= 0:
        path.append(last)
        last = parents[last]
    return path[::-1]


def _seen(p, length, left, sinks):
    """How many of the `length` keys before a draft the query at position p sees."""
    first = min(length, max(0, p - left)) if left >= 0 else 0
    return length - first + min(sinks, first)


def work(case):
    c = case
    if c["kind"] == "rotate":
        n = sum(_spread(c["batch"], c["low"], c["high"]))
        return {"bytes": 2 * n * (c["heads"] + c["kv_heads"]) * c["head_dim"] * _BYTES[c["dtype"]], "flops": 3 * n * (c["heads"] + c["kv_heads"]) * c["dims"]}
    new = _spread(c["batch"], c["new_low"], c["new_high"])
    if c["kind"] == "append":
        e, ce, n = _BYTES[c["dtype"]], _BYTES[c["cache"]], sum(new)
        return {"bytes": n * c["head_dim"] * (2 * c["heads"] * e + 2 * c["kv_heads"] * (e + ce)), "flops": 3 * n * (c["heads"] + c["kv_heads"]) * c["dims"]}
    if c["kind"] == "tree":
        return {"bytes": sum(new) * 4 * (2 + -(-c["new_high"] // 32)), "flops": 0}
    old = _spread(c["batch"], c["low"], c["high"])
    if c["kind"] == "verify":
        pairs = rows = 0
        for n, o in zip(new, old):
            depths = _depths(_parents(n, c["width"]))
            for d in depths:
                pairs += _seen(o + d, o, c["left"], c["sinks"]) + (d + 1 if c["left"] < 0 else min(d, c["left"]) + 1)
            rows += n + _seen(o, o, c["left"], c["sinks"])
        kv = 2 * rows * c["kv_heads"] * c["head_dim"] * _BYTES[c["cache"]]
        return {"bytes": kv + 2 * sum(new) * c["heads"] * c["head_dim"] * _BYTES[c["dtype"]] + 4 * rows // c["page_tokens"], "flops": 4 * c["head_dim"] * c["heads"] * pairs}
    moved = gone = 0
    for n, o, last in zip(new, old, _last(c)):
        path = _path(_parents(n, c["width"]), last)
        moved += sum(1 for j, p in enumerate(path) if p != j)
        gone += -(-(o + n) // c["page_tokens"]) - -(-(o + len(path)) // c["page_tokens"])
    row = 2 * c["layers"] * c["kv_heads"] * c["head_dim"] * _BYTES[c["cache"]]
    return {"bytes": 2 * moved * row + 16 * c["batch"] + 12 * gone + 4 * c["batch"] * -(-c["new_high"] // 32), "flops": 0}


# ------------------------------------------------------------------------------------------------ what a program has in hand

def _rand(gen, *shape, dtype=torch.float32):
    return torch.randn(shape, device="cuda", generator=gen, dtype=torch.float32 if dtype == torch.float32 else torch.float16).to(dtype)


def _ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def _starts(counts):
    at = [0]
    for n in counts:
        at.append(at[-1] + n)
    return _ints(at)


def _tables(gen, lens, page_tokens, pages, width):
    """Each sequence's pages, anywhere in the cache."""
    order, at, rows = torch.randperm(pages, generator=gen, device="cuda").tolist(), 0, []
    for n in lens:
        k = -(-n // page_tokens)
        rows.append(order[at:at + k] + [-1] * (width - k))
        at += k
    return _ints(rows)


def _freqs(c):
    """Radians a position of each pair"""
    return c["base"] ** (-torch.arange(0, c["dims"], 2, dtype=torch.float64, device="cuda") / c["dims"])


def prepare(case, seed):
    c = case
    gen = torch.Generator(device="cuda").manual_seed(seed)
    if c["kind"] == "rotate":
        lens, dt = _spread(c["batch"], c["low"], c["high"]), _DTYPES[c["dtype"]]
        n, d, kd = sum(lens), c["heads"] * c["head_dim"], c["kv_heads"] * c["head_dim"]
        return {**c, "qkv": _rand(gen, n, d + 2 * kd, dtype=dt), "q_out": torch.zeros(n, d, device="cuda", dtype=dt), "k_out": torch.zeros(n, kd, device="cuda", dtype=dt),
                "starts": _starts(lens), "freqs": _freqs(c)}
    new = _spread(c["batch"], c["new_low"], c["new_high"])
    s = {**c, "starts": _starts(new)}
    if c["kind"] == "tree" or c["width"] >= 0:
        words = -(-c["new_high"] // 32)
        s["parents"] = _ints([p for n in new for p in _parents(n, c["width"])])
        s["masks"] = torch.zeros(sum(new), words, device="cuda", dtype=torch.int32)
        s["depths"] = torch.zeros(sum(new), device="cuda", dtype=torch.int32)
    if c["kind"] == "tree":
        # each seed has drafts of its own: nodes hang one before or one after where they would, among those before them
        shift = torch.randint(0, 2, s["parents"].shape, generator=gen, device="cuda", dtype=torch.int32)
        s["parents"] = torch.maximum(s["parents"] - shift, torch.full_like(s["parents"], -1))
        return s
    if "masks" in s:
        s["masks"].copy_(_plain_tree(s)[0])
        s["depths"].copy_(_plain_tree(s)[1])
    old, ct, pt = _spread(c["batch"], c["low"], c["high"]), _DTYPES[c["cache"]], c["page_tokens"]
    lens = [a + b for a, b in zip(new, old)]
    need = sum(-(-x // pt) for x in lens)
    pages, width = need + need // 8 + 1, -(-max(lens) // pt)
    s |= {"lengths": _ints(lens), "tables": _tables(gen, lens, pt, pages, width), "refs": torch.zeros(pages, dtype=torch.int32, device="cuda")}
    s["refs"][s["tables"][s["tables"] >= 0].long()] = 1
    for name in ("k_pages", "v_pages"):
        s[name] = _rand(gen, c.get("layers", 1), pages, c["kv_heads"], pt, c["head_dim"], dtype=ct)
    if c["kind"] == "accept":
        s["last"], s["kept"] = _ints(_last(c)), torch.zeros(c["batch"], dtype=torch.int32, device="cuda")
        s |= {"long_" + name: s[name].clone() for name in ("tables", "lengths", "refs")}
        return s
    dt, d, kd = _DTYPES[c["dtype"]], c["heads"] * c["head_dim"], c["kv_heads"] * c["head_dim"]
    s["q"], s["out"] = _rand(gen, sum(new), d, dtype=dt), torch.zeros(sum(new), d, device="cuda", dtype=dt)
    s["max_new"] = max(new)
    if c["kind"] == "append":
        s["k"], s["v"] = (_rand(gen, sum(new), kd, dtype=dt) for _ in range(2))
        s["freqs"] = _freqs(c)
    return s


# ------------------------------------------------------------------------------------------------ one pass

def _ctx():
    """One context for the process, as a serving program holds it: on the stream that torch is on at the first pass, on which the program stays.  Torch's default stream has no
    handle (0), and the context keeps its own stream then, which takes turns with the default one: so a pass that changes from torch's work to the library's, or back, waits for it."""
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


def _handles(s):
    """The program's handles of its cache, rotation and trees."""
    if "handles" not in s:
        ctx, h = _ctx(), {}
        if "tables" in s:
            h["cache"] = _pages.PagedCache.over(ctx, _package, s["k_pages"], s["v_pages"], s["tables"], s["lengths"], s["refs"])
        if "freqs" in s:
            h["rotary"] = _pages.Rotary(ctx, _package, s["head_dim"], pairs=s["pairs"], freqs=s["freqs"])
        h["tree"] = _pages.DraftTree.over(ctx, _package, s["masks"], s["depths"]) if "masks" in s else None
        s["handles"] = h
    return s["handles"]


def run(state):
    return {"rotate": _run_rotate, "append": _run_append, "tree": _run_tree, "verify": _run_verify, "accept": _run_accept}[state["kind"]](state)


def _sequence_of(starts, n):
    """Of each of n packed tokens: its row of the batch, and its place among that row's tokens"""
    at = torch.arange(n, device=starts.device)
    seq = torch.searchsorted(starts[1:].contiguous(), at, right=True)
    return seq, at - starts.long()[seq]


def _turned(x, position, freqs, dims, pairs, head_dim):
    """x [tokens][columns] turned by its tokens' positions, in fp32; angles in 64 bits"""
    angle = position.double()[:, None] * freqs
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]
    y = x.float().unflatten(-1, (-1, head_dim))
    turn = y[..., :dims]
    a, b = (turn[..., :dims // 2], turn[..., dims // 2:]) if pairs == "halves" else (turn[..., 0::2], turn[..., 1::2])
    out = (a * cos - b * sin, a * sin + b * cos)
    turn = torch.cat(out, -1) if pairs == "halves" else torch.stack(out, -1).flatten(-2)
    return torch.cat((turn, y[..., dims:]), -1).flatten(1)


def _run_rotate(s):
    d, kd, qkv = s["heads"] * s["head_dim"], s["kv_heads"] * s["head_dim"], s["qkv"]
    q, k, q_out, k_out = qkv[:, :d], qkv[:, d:d + kd], s["q_out"], s["k_out"]
    if own:
        _handles(s)["rotary"].rotate(q, k, q_out, k_out, s["starts"])
        return q_out, k_out
    _, place = _sequence_of(s["starts"], qkv.shape[0])
    for x, out in ((q, q_out), (k, k_out)):
        out.copy_(_turned(x, place, s["freqs"], s["dims"], s["pairs"], s["head_dim"]).to(out.dtype))
    return q_out, k_out


def _run_append(s):
    k_pages, v_pages, out = s["k_pages"], s["v_pages"], s["out"]
    if own:
        h = _handles(s)
        h["cache"].append(0, s["k"], s["v"], s["starts"], rotary=h["rotary"], q=s["q"], q_out=out, tree=h["tree"])
        return k_pages, v_pages, out
    pt, n = s["page_tokens"], s["k"].shape[0]
    seq, place = _sequence_of(s["starts"], n)
    before = (s["lengths"] - (s["starts"][1:] - s["starts"][:-1])).long()[seq]
    position, slot = before + (s["depths"].long() if "depths" in s else place), before + place
    page = s["tables"].long()[seq, slot // pt]
    turn = (position, s["freqs"], s["dims"], s["pairs"], s["head_dim"])
    out.copy_(_turned(s["q"], *turn).to(out.dtype))
    for pool, x in ((k_pages, _turned(s["k"], *turn)), (v_pages, s["v"])):
        pool[0][page, :, slot % pt] = x.unflatten(-1, (s["kv_heads"], s["head_dim"])).to(pool.dtype)
    return k_pages, v_pages, out


def _plain_tree(s):
    """(masks, depths): who is whose ancestor by squaring the relation 'is or is the parent of' until it holds over any distance"""
    starts, parents, words = s["starts"], s["parents"], s["masks"].shape[1]
    seq, place = _sequence_of(starts, parents.shape[0])
    rel = torch.eye(32 * words, device=parents.device).repeat(starts.shape[0] - 1, 1, 1)
    child = parents >= 0
    rel[seq[child], place[child], parents[child].long()] = 1.0
    for _ in range((32 * words - 1).bit_length()):
        rel = (torch.bmm(rel, rel) > 0).float()
    rows = rel[seq, place]
    bits = rows.long().unflatten(-1, (words, 32)) << torch.arange(32, device=parents.device)
    return bits.sum(-1).int(), (rows.sum(-1) - 1).int()


def _run_tree(s):
    masks, depths = s["masks"], s["depths"]
    if own:
        _handles(s)["tree"].build(s["parents"], s["starts"])
        return masks, depths
    m, d = _plain_tree(s)
    masks.copy_(m)
    depths.copy_(d)
    return masks, depths


def _unpacked(masks):
    """[tokens][words] as truth values [tokens][32 * words]"""
    return ((masks[..., None] >> torch.arange(32, device=masks.device)) & 1).flatten(1).bool()


def _run_verify(s):
    h, kv, hd, pt, out, starts, lengths = s["heads"], s["kv_heads"], s["head_dim"], s["page_tokens"], s["out"], s["starts"], s["lengths"]
    if own:
        t = _handles(s)
        t["cache"].attend(0, s["q"], out, starts, h, left=s["left"] if s["left"] >= 0 else None, sinks=s["sinks"], tree=t["tree"])
        return out
    most, batch = s["max_new"], s["batch"]
    at = torch.arange(most, device=out.device)
    here = at[None, :] < (starts[1:] - starts[:-1])[:, None]
    rows = torch.where(here, starts[:-1, None] + at, 0).long()
    before = lengths - (starts[1:] - starts[:-1])
    key = torch.arange(s["tables"].shape[1] * pt, device=out.device)
    held = key[None, :] < lengths[:, None]
    node = key[None, :] - before[:, None]  # which node of its tree a key is; negative: it was there before
    k_node = node.clamp(0, most - 1).long()
    position = torch.where(node < 0, key[None, :], before[:, None] + s["depths"][rows.gather(1, k_node)])
    mine = before[:, None] + s["depths"][rows]  # [batch][most]
    kin = _unpacked(s["masks"])[rows].gather(2, k_node[:, None, :].expand(-1, most, -1))
    seen = held[:, None, :] & ((node < 0)[:, None, :] | kin) & here[:, :, None]
    if s["left"] >= 0:
        seen &= (position[:, None, :] + s["left"] >= mine[:, :, None]) | (position < s["sinks"])[:, None, :]
    pages = s["tables"].clamp(min=0).long()
    k, v = (x[0][pages].float().permute(0, 2, 1, 3, 4).reshape(batch * kv, -1, hd) for x in (s["k_pages"], s["v_pages"]))
    v = torch.where(held.repeat_interleave(kv, 0)[:, :, None], v, 0.0)
    q = s["q"][rows].float().reshape(batch, most, kv, h // kv, hd).permute(0, 2, 3, 1, 4).reshape(batch * kv, h // kv * most, hd)
    score = torch.bmm(q, k.transpose(1, 2).contiguous()).mul_(1 / math.sqrt(hd)).reshape(batch, kv, h // kv, most, -1)
    score.masked_fill_(~seen[:, None, None], -math.inf)
    top = score.amax(-1, keepdim=True)
    score = score.sub_(torch.where(top == -math.inf, 0.0, top)).exp_()
    total = score.sum(-1, keepdim=True)
    o = torch.bmm(score.reshape(batch * kv, h // kv * most, -1), v).reshape(batch, kv, h // kv, most, hd) / torch.where(total > 0, total, 1.0)
    out[rows[here]] = o.permute(0, 3, 1, 2, 4).reshape(batch, most, h * hd)[here].to(out.dtype)
    return out


def _run_accept(s):
    tables, lengths, refs, kept = s["tables"], s["lengths"], s["refs"], s["kept"]
    for name in ("tables", "lengths", "refs"):  # (as the next draft came)
        s[name].copy_(s["long_" + name])
    if own:
        h = _handles(s)
        h["cache"].accept(h["tree"], s["last"], kept, s["starts"])
        return s["k_pages"], s["v_pages"], tables, lengths, refs, kept
    pt, starts, last = s["page_tokens"], s["starts"], s["last"].long()
    before = lengths - (starts[1:] - starts[:-1])
    bits = _unpacked(s["masks"])[(starts[:-1] + last.clamp(min=0)).long()] & (last >= 0)[:, None]
    count = bits.sum(-1)
    kept.copy_(count)
    path = torch.sort((~bits).int(), dim=-1, stable=True)[1]  # the branch's nodes first, in their order
    step = torch.arange(bits.shape[1], device=bits.device)
    b, j = torch.nonzero(step[None, :] < count[:, None], as_tuple=True)
    src, dst = before[b] + path[b, j], before[b] + j
    sp, dp = tables[b, src // pt].long(), tables[b, dst // pt].long()
    for pool in (s["k_pages"], s["v_pages"]):
        pool[:, dp, :, dst % pt] = pool[:, sp, :, src % pt]
    lengths.copy_(before + count)
    gone = torch.arange(tables.shape[1], device=tables.device)[None, :] >= ((lengths + pt - 1) // pt)[:, None]
    free = tables[gone & (tables >= 0)].long()
    refs.index_add_(0, free, -torch.ones_like(free, dtype=torch.int32))
    tables.masked_fill_(gone, -1)
    return s["k_pages"], s["v_pages"], tables, lengths, refs, kept


# ------------------------------------------------------------------------------------------------ the definition in 64 bits

def exact(case, seed):
    if case["kind"] in ("tree", "accept"):
        return None  # whole numbers, and rows that are moved as they are
    s = prepare(case, seed)
    if case["kind"] == "verify":
        return _exact_verify(s)
    d, kd, at = s["heads"] * s["head_dim"], s["kv_heads"] * s["head_dim"], s["starts"].tolist()
    if case["kind"] == "rotate":
        place = torch.cat([torch.arange(b - a, device="cuda") for a, b in zip(at, at[1:])])
        return _exact_turned(s, s["qkv"][:, :d], place), _exact_turned(s, s["qkv"][:, d:d + kd], place)
    pools, turned, lens = [s["k_pages"].double(), s["v_pages"].double()], [], s["lengths"].tolist()
    for b in range(s["batch"]):
        rows, old = slice(at[b], at[b + 1]), lens[b] - (at[b + 1] - at[b])
        slot = torch.arange(old, lens[b], device="cuda")
        place = slot if s["width"] < 0 else old + torch.tensor(_depths(_parents(lens[b] - old, s["width"])), device="cuda")
        turned.append(_exact_turned(s, s["q"][rows], place))
        page = s["tables"][b].long()[slot // s["page_tokens"]]
        for pool, x in zip(pools, (_exact_turned(s, s["k"][rows], place), s["v"][rows].double())):
            pool[0, page, :, slot % s["page_tokens"]] = x.reshape(-1, s["kv_heads"], s["head_dim"])
    return pools[0], pools[1], torch.cat(turned)


def _exact_turned(s, x, place):
    """As a complex number, each pair times e^(i p f)"""
    y = x.double().reshape(x.shape[0], -1, s["head_dim"]).clone()
    half, n = s["dims"] // 2, s["dims"]
    first, second = (slice(0, half), slice(half, n)) if s["pairs"] == "halves" else (slice(0, n, 2), slice(1, n, 2))
    z = torch.complex(y[..., first].contiguous(), y[..., second].contiguous()) * torch.polar(torch.ones_like(s["freqs"]), s["freqs"] * place[:, None].double())[:, None]
    y[..., first], y[..., second] = z.real, z.imag
    return y.reshape(x.shape)


def _exact_verify(s):
    """Sequence by sequence, key head by key head: softmax(q k^T / sqrt(hd)) v over the keys that each node sees."""
    h, kv, hd, at = s["heads"], s["kv_heads"], s["head_dim"], s["starts"].tolist()
    out = torch.zeros(at[-1], h, hd, device="cuda", dtype=torch.float64)
    for b, length in enumerate(s["lengths"].tolist()):
        n = at[b + 1] - at[b]
        old, parents = length - n, _parents(n, s["width"])
        depth = torch.tensor(_depths(parents), device="cuda")
        kin = torch.zeros(n, n, dtype=torch.bool)
        for i in range(n):
            kin[i, _path(parents, i)] = True
        seen = torch.cat((torch.ones(n, old, dtype=torch.bool, device="cuda"), kin.cuda()), 1)
        if s["left"] >= 0:
            where = torch.cat((torch.arange(old, device="cuda"), old + depth))
            seen &= ((old + depth)[:, None] - where[None, :] <= s["left"]) | (where < s["sinks"])[None, :]
        page = s["tables"][b, :-(-length // s["page_tokens"])].long()
        k, v = (x[0, page].transpose(1, 2).reshape(-1, kv, hd)[:length].double() for x in (s["k_pages"], s["v_pages"]))
        q = s["q"][at[b]:at[b + 1]].double().reshape(n, kv, h // kv, hd)
        for a in range(kv):
            score = (q[:, a].reshape(-1, hd) @ k[:, a].t().contiguous()).reshape(n, h // kv, length) / math.sqrt(hd)
            share = torch.softmax(score.masked_fill(~seen[:, None], -math.inf), -1)
            out[at[b]:at[b + 1], a * (h // kv):(a + 1) * (h // kv)] = (share.reshape(-1, length) @ v[:, a].contiguous()).reshape(n, h // kv, hd)
    return out.reshape(at[-1], h * hd)
