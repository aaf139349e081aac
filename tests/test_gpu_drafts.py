"""Rotated positions, trees of drafted tokens, attention of them over a paged cache and accepting a branch, on the GPU, against plain float64 (rotation, attention) and sequential
models (trees, pages).

Tolerances of the rotation.  With u = 2^-24: the angle that is left after whole quarter turns, at most pi / 4, is rounded to fp32 once (0.8 u) and evaluated by polynomials whose last
step rounds to u and whose inner ones add less than u: a sine or cosine is within 3 u, counting the cut-off of the series (2e-9, 0.04 u), and within 2^-52 of the angle, which
is a rounded product in 64 bits.  a cos - b sin has one product rounded on its own (u |b|) and one rounding of the sum (u (|a| + |b|)).  So a result is within
(5 u + angle 2^-52) (|a| + |b|), and half a step of the output's type (subnormal numbers: of the smallest one).

Tolerances of attention: those of the cache's attention, whose sums are the same; the keys that a node does not see are no part of them."""
import math

import numpy as np
import pytest
import torch

from __graft_entry__ import load_package
from test_gpu_serving import HALF, PAIRS, TYPES, U, Filled, check, check_pieces, gen_of, ints, plan_is, randn, small_cache, starts_of
from test_gpu_serving import _model as unrotated_model

pimdl = load_package()
from pim_dl_asplos_amd import kvcache as K  # noqa: E402

pytestmark = pytest.mark.gpu
TINY = {"f32": 2.0 ** -149, "f16": 2.0 ** -25, "bf16": 2.0 ** -134}


@pytest.fixture(scope="module")
def ctx():
    c = pimdl.Context(0)
    c.set_stream(torch.cuda.current_stream().cuda_stream)
    yield c
    c.close()


# ---------------------------------------------------------------------------------------------- rotation

def turned(x, place, freqs, pairs, hd):
    """x [n][columns] turned by `place` in 64 bits: (values, (|a| + |b|) (5 u + angle 2^-52))"""
    y = x.double().reshape(x.shape[0], -1, hd)
    half = freqs.shape[0]
    angle = place.double()[:, None] * freqs
    c, s = angle.cos()[:, None], angle.sin()[:, None]
    first, second = (slice(0, half), slice(half, 2 * half)) if pairs == "halves" else (slice(0, 2 * half, 2), slice(1, 2 * half, 2))
    a, b, out, off = y[..., first], y[..., second], y.clone(), torch.zeros_like(y)
    out[..., first], out[..., second] = a * c - b * s, a * s + b * c
    off[..., first] = off[..., second] = (a.abs() + b.abs()) * (5 * U + angle.abs()[:, None] * 2.0 ** -52)
    return out.reshape(x.shape), off.reshape(x.shape)


def check_turned(got, want, off, dtype):
    tol = off + HALF[dtype] * (want.abs() + off) + TINY[dtype]
    bad = ~((got.double() - want).abs() <= tol)
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()}, worst {float(((got.double() - want).abs() / tol).max()):.2f} of the tolerance"


def rotary_of(ctx, hd, dims, pairs, base=10000.0):
    return K.Rotary(ctx, pimdl, hd, base=base, dims=dims, pairs=pairs)


def places_of(counts):
    return torch.cat([torch.arange(c, device="cuda") for c in counts])


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("pairs", ["halves", "neighbours"])
@pytest.mark.parametrize("counts,heads,kv,hd,dims", [
    ([1], 1, 1, 2, 2),                        # the smallest
    ([5, 1, 0, 70], 4, 2, 64, 64),
    ([128], 12, 12, 64, 64),
    ([300, 17], 32, 8, 128, 128),
    ([33], 3, 1, 80, 40),                     # half of a head's columns
    ([40, 9], 2, 2, 96, 20),                  # packs of four
    ([21, 2], 5, 1, 31, 30),                  # an odd head: a column is left over
    ([19], 2, 3, 7, 2),
    ([50], 0, 2, 64, 64),                     # keys alone
    ([50], 2, 0, 64, 64),                     # queries alone
    ([7, 3], 48, 48, 256, 256),               # more units to a token than threads
    ([3], 100, 1, 63, 62),
    ([2] * 700, 1, 1, 32, 32),                # many sequences: not every start in shared memory ...
    ([1, 0, 2] * 1100, 1, 1, 16, 16),         # ... nor every second one
])
def test_rotate_against_float64(ctx, dtype, pairs, counts, heads, kv, hd, dims):
    r, n, d, kd, gen = rotary_of(ctx, hd, dims, pairs), sum(counts), heads * hd, kv * hd, gen_of(hd + dims)
    extra = 8 if hd % 8 == 0 else 3
    buf = randn(gen, n + 3, d + kd + extra, dtype=dtype)
    q_out, k_out = (torch.full((n + 3, w + extra), -5.0, device="cuda", dtype=TYPES[dtype]) for w in (d, kd))
    r.rotate(buf[:, :d], buf[:, d:d + kd], q_out[:, :d], k_out[:, :kd], starts_of(counts))
    torch.cuda.synchronize()
    for out, x, w in ((q_out, buf[:, :d], d), (k_out, buf[:, d:d + kd], kd)):
        assert (out[n:] == -5.0).all() and (out[:, w:] == -5.0).all()  # rows behind the last sequence, columns behind the heads
        want, off = turned(x[:n], places_of(counts), r.freqs, pairs, hd)
        check_turned(out[:n, :w], want, off, dtype)
        left = torch.arange(w, device="cuda") % hd >= dims
        assert torch.equal(out[:n, :w][:, left], x[:n][:, left])
    before = buf.clone()
    r.rotate(buf[:, :d], buf[:, d:d + kd], buf[:, :d], buf[:, d:d + kd], starts_of(counts))  # in place: the same, bit for bit
    torch.cuda.synchronize()
    assert torch.equal(buf[:n, :d], q_out[:n, :d]) and torch.equal(buf[:n, d:d + kd], k_out[:n, :kd])
    assert torch.equal(buf[n:], before[n:]) and torch.equal(buf[:, d + kd:], before[:, d + kd:])


@pytest.mark.parametrize("shift", [1, 2, 4])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_rotate_at_any_alignment(ctx, dtype, shift):
    """Rows that begin anywhere and have any stride: the same numbers as aligned ones."""
    r, n, d = rotary_of(ctx, 64, 64, "halves"), 37, 4 * 64
    wide = randn(gen_of(1), n, 2 * d + 16 + shift, dtype=dtype)
    q, k = wide[:, shift:shift + d], wide[:, shift + d:shift + 2 * d]
    out = [torch.zeros(n, d, device="cuda", dtype=TYPES[dtype]) for _ in range(4)]
    r.rotate(q, k, out[0], out[1], starts_of([20, 17]))
    r.rotate(q.contiguous(), k.contiguous(), out[2], out[3], starts_of([20, 17]))
    torch.cuda.synchronize()
    assert torch.equal(out[0], out[2]) and torch.equal(out[1], out[3])


@pytest.mark.parametrize("pairs", ["halves", "neighbours"])
def test_rotate_by_given_positions_near_and_far(ctx, pairs):
    """Positions before the first, on both sides of quarter turns, and up to the ends of 32 bits."""
    hd, quarter = 8, [round(i * math.pi / 2) for i in range(-9, 10)]
    place = torch.tensor([0, -1, 1, -2 ** 31, 2 ** 31 - 1, 1 << 30, 123456789, -987654321, 131071, 65536] + quarter, dtype=torch.int32, device="cuda")
    n = place.shape[0]
    freqs = torch.tensor([1.0, 2.0, 0.25, 1e-9], dtype=torch.float64, device="cuda")
    r = K.Rotary(ctx, pimdl, hd, pairs=pairs, freqs=freqs)
    x = randn(gen_of(2), n, 3 * hd)
    out = torch.zeros_like(x)
    r.rotate(x, x[:, :0], out, out[:, :0], starts_of([n]), positions=place)
    torch.cuda.synchronize()
    want, off = turned(x, place, freqs, pairs, hd)
    check_turned(out, want, off, "f32")
    r.rotate(x, x[:, :0], out, out[:, :0], starts_of([5, n - 5]), positions=torch.zeros_like(place))
    torch.cuda.synchronize()
    assert torch.equal(out, x)  # nothing turns at position 0


def test_rotate_keeps_infinities_and_nans_to_their_pairs(ctx):
    r, x = rotary_of(ctx, 64, 32, "halves"), randn(gen_of(3), 4, 128)
    x[1, 3], x[2, 70], x[3, 40] = float("inf"), float("nan"), float("-inf")
    out = torch.zeros_like(x)
    r.rotate(x, x[:, :0], out, out[:, :0], starts_of([4]))
    torch.cuda.synchronize()
    bad = ~torch.isfinite(out)
    want = torch.zeros_like(bad)
    want[1, [3, 19]] = want[2, [70, 86]] = True
    want[3, 40] = True
    assert torch.equal(bad, want) and out[3, 40] == float("-inf")


def test_rotate_beyond_one_row_of_workgroups(ctx):
    n = (1 << 26) + 100  # 64 tokens to a workgroup, 2^20 of them in a row
    r = rotary_of(ctx, 2, 2, "neighbours")
    x = torch.ones(n, 2, device="cuda", dtype=torch.bfloat16)
    r.rotate(x, x[:, :0], x, x[:, :0], ints(0, 70, n - 1, n))
    torch.cuda.synchronize()
    for lo, hi, base in ((0, 70, 0), (70, 400, 70), ((1 << 26) - 50, (1 << 26) + 99, 70), (n - 1, n, n - 1)):
        place = torch.arange(lo - base, hi - base, device="cuda")
        want, off = turned(torch.ones(hi - lo, 2, device="cuda"), place, r.freqs, "neighbours", 2)
        check_turned(x[lo:hi], want, off, "bf16")


# ---------------------------------------------------------------------------------------------- append with a rotation

@pytest.mark.parametrize("dtype,cache", PAIRS)
@pytest.mark.parametrize("counts,lengths,heads,kv,hd,dims,pairs,page_tokens,tree", [
    ([1], [1], 1, 1, 64, 64, "halves", 16, False),
    ([1, 1, 1], [1, 16, 17], 12, 12, 64, 16, "halves", 16, False),
    ([70, 0, 33], [70, 5, 100], 8, 2, 80, 80, "neighbours", 32, False),
    ([20, 3], [30, 2], 3, 3, 17, 16, "halves", 16, False),      # more tokens than positions: the first ones have no place
    ([200], [333], 32, 8, 128, 128, "halves", 64, False),
    ([9, 40, 1], [60, 41, 1], 4, 2, 64, 64, "neighbours", 16, True),
    ([33, 100], [500, 1000], 6, 3, 96, 40, "halves", 128, True),
    ([5, 6], [50, 60], 0, 2, 64, 64, "halves", 16, False),      # keys without queries
])
def test_append_turns_rounds_and_places(ctx, dtype, cache, counts, lengths, heads, kv, hd, dims, pairs, page_tokens, tree):
    f, n, gen = Filled(ctx, sum(lengths), lengths, kv, hd, page_tokens, cache), sum(counts), gen_of(3)
    c, r = f.cache, rotary_of(ctx, hd, dims, pairs)
    buf = randn(gen, n + 2, (heads + 2 * kv) * hd + 8, dtype=dtype, scale=3.0)
    q, k, v = buf[:n, :heads * hd], buf[:n, heads * hd:(heads + kv) * hd], buf[:n, (heads + kv) * hd:(heads + 2 * kv) * hd]
    t, depths = None, places_of(counts)
    if tree:
        parents = forest(counts, 7)
        t = K.DraftTree(ctx, pimdl, n, most=max(counts))
        t.build(parents, starts_of(counts))
        depths = torch.tensor(np.concatenate([depths_of(p) for p in split(parents, counts)]), device="cuda")
    base = torch.tensor(np.repeat(np.array(lengths) - np.array(counts), counts), device="cuda")
    want_k, off_k = turned(k, base + depths, r.freqs, pairs, hd)
    pools = [x.clone() for x in (c.k, c.v)]
    q_out = torch.full((n + 2, heads * hd), -5.0, device="cuda", dtype=TYPES[dtype])
    c.append(0, k, v, starts_of(counts), rotary=r, q=q if heads else None, q_out=q_out[:n], tree=t)
    torch.cuda.synchronize()
    assert (q_out[n:] == -5.0).all()
    if heads:
        want, off = turned(q, base + depths, r.freqs, pairs, hd)
        check_turned(q_out[:n], want, off, dtype)
    at = 0
    for s, m in enumerate(counts):
        for i in range(m):
            pos = lengths[s] - m + i
            if pos < 0:
                continue
            page, row = int(c.tables[s, pos // page_tokens]), pos % page_tokens
            check_turned(c.k[0, page, :, row].flatten(), want_k[at + i], off_k[at + i], cache)
            assert torch.equal(c.v[0, page, :, row].flatten(), v[at + i].to(TYPES[cache]))
            for pool, old in zip((c.k, c.v), pools):
                old[0, page, :, row] = pool[0, page, :, row]
        at += m
    bits = torch.int32 if cache == "f32" else torch.int16
    for pool, old in zip((c.k, c.v), pools):  # everywhere else: as it was
        assert torch.equal(pool.view(bits), old.view(bits))


def test_append_turned_in_place_and_by_lists(ctx):
    """Queries turned where they are; the rows of the batch are those sequences that `seqs` names, one of them not there."""
    f, r = Filled(ctx, 8, [64, 100, 7], 2, 64, 16, "f16"), rotary_of(ctx, 64, 64, "halves")
    x = randn(gen_of(9), 6, 8 * 64)
    q, k, v, raw = x[:, :256], x[:, 256:384], x[:, 384:], x[:, :256].clone()
    before = f.cache.k.clone()
    f.cache.append(0, k, v, starts_of([2, 1, 3]), ints(2, 77, 1), rotary=r, q=q, q_out=q)
    torch.cuda.synchronize()
    place = torch.tensor([5, 6, -1, 97, 98, 99], device="cuda")
    want, off = turned(raw, place, r.freqs, "halves", 64)
    check_turned(q, want, off, "f32")
    want, off = turned(k, place, r.freqs, "halves", 64)
    for row, s in ((0, 2), (1, 2), (3, 1), (4, 1), (5, 1)):
        page, at = int(f.cache.tables[s, int(place[row]) // 16]), int(place[row]) % 16
        check_turned(f.cache.k[0, page, :, at].flatten(), want[row], off[row], "f16")
        before[0, page, :, at] = f.cache.k[0, page, :, at]
    assert torch.equal(f.cache.k.view(torch.int16), before.view(torch.int16))


def test_append_turned_without_room_or_pages_writes_no_keys(ctx):
    """Where the last reserve lacked pages, and where a table's entry is no page; the queries are turned all the same."""
    cache, r = small_cache(ctx, 5, pages=3, seqs=2, width=8), rotary_of(ctx, 16, 16, "neighbours")
    cache.reserve(ints(0), ints(40))
    cache.reserve(ints(0), ints(20))
    assert int(cache.lacking) == 1
    before, x, out = cache.k.clone(), randn(gen_of(1), 20, 32), torch.zeros(20, 32, device="cuda")
    cache.append(0, x, x, starts_of([20]), ints(0), rotary=r, q=x, q_out=out)
    torch.cuda.synchronize()
    assert torch.equal(cache.k, before)
    want, off = turned(x, torch.arange(20, 40, device="cuda"), r.freqs, "neighbours", 16)
    check_turned(out, want, off, "f32")
    f = Filled(ctx, 3, [40], 1, 64, 16, "f16", width=3)
    f.cache.tables[0, 1], f.cache.tables[0, 2] = -1, 1 << 20
    before, x, r = f.cache.k.clone(), randn(gen_of(1), 40, 64), rotary_of(ctx, 64, 64, "halves")
    f.cache.append(0, x, x, starts_of([40]), rotary=r)
    torch.cuda.synchronize()
    page = int(f.cache.tables[0, 0])
    assert torch.equal(f.cache.v[0, page, 0], x[:16].half())
    before[0, page] = f.cache.k[0, page]
    assert torch.equal(f.cache.k.view(torch.int16), before.view(torch.int16))


def test_append_turned_at_two_thousand_million(ctx):
    """The newest tokens of a sequence of 2 000 000 000 positions, whose older pages are gone."""
    length, pt = 2_000_000_000, 1024
    tables = torch.full((1, -(-length // pt)), -1, device="cuda", dtype=torch.int32)
    tables[0, -1], tables[0, -2] = 0, 1
    pools = [torch.zeros(1, 2, 2, pt, 64, device="cuda") for _ in range(2)]
    c = K.PagedCache.over(ctx, pimdl, *pools, tables, ints(length), ints(1, 1))
    r, x, out = rotary_of(ctx, 64, 64, "halves"), randn(gen_of(4), 9, 128), torch.zeros(9, 128, device="cuda")
    c.append(0, x, x, starts_of([9]), rotary=r, q=x, q_out=out)
    torch.cuda.synchronize()
    want, off = turned(x, torch.arange(length - 9, length, device="cuda"), r.freqs, "halves", 64)
    check_turned(out, want, off, "f32")
    for i, pos in enumerate(range(length - 9, length)):
        assert torch.equal(pools[0][0, int(tables[0, pos // pt]), :, pos % pt].flatten(), out[i])


# ---------------------------------------------------------------------------------------------- trees

def split(parents, counts):
    at, out = 0, []
    p = parents.tolist()
    for c in counts:
        out.append(p[at:at + c])
        at += c
    return out


def forest(counts, seed, width=None):
    """Random trees: each node hangs on one before it or on none; width: chains side by side (see test_chains)."""
    rng = np.random.default_rng(seed)
    if width:
        return ints(*[-1 if i == 0 else 0 if i <= width else i - width for c in counts for i in range(c)])
    return ints(*[int(rng.integers(-1, i)) if i else -1 for c in counts for i in range(c)])


def depths_of(parents):
    d = []
    for p in parents:
        d.append(0 if p < 0 else d[p] + 1)
    return d


def kin_of(parents):
    """[n][n]: which node is which node's ancestor, or itself"""
    n = len(parents)
    kin = np.zeros((n, n), bool)
    for i, p in enumerate(parents):
        if p >= 0:
            kin[i] = kin[p]
        kin[i, i] = True
    return kin


def words_of(kin, words):
    n = kin.shape[0]
    wide = np.zeros((n, 32 * words), np.uint64)
    wide[:, :n] = kin
    return (wide.reshape(n, words, 32) << np.arange(32, dtype=np.uint64)).sum(-1).astype(np.uint32).view(np.int32)


@pytest.mark.parametrize("most", [1, 2, 31, 32, 33, 64, 65, 96, 100, 128, 129, 200, 256, 257, 500, 512, 513, 700, 1023, 1024])
def test_trees_against_a_sequential_model(ctx, most):
    """Random trees, one chain, chains side by side, nothing but roots, trees of one node and of none; rows behind the last tree."""
    counts = [most, 1, 0, max(1, most // 2), most, most, most]
    some = [most, 1, 0, max(1, most // 2)]
    parents = torch.cat([forest(some, most), ints(*range(-1, most - 1)), forest([most], 1, width=3), ints(*[-1] * most)])
    n, words = sum(counts), -(-most // 32)
    tree = K.DraftTree.over(ctx, pimdl, torch.full((n + 2, words), -5, device="cuda", dtype=torch.int32), torch.full((n + 2,), -5, device="cuda", dtype=torch.int32))
    tree.build(torch.cat([parents, ints(0, 0)]), starts_of(counts))
    torch.cuda.synchronize()
    assert (tree.masks[n:] == -5).all() and (tree.depths[n:] == -5).all()
    masks, depths = tree.masks.cpu().numpy(), tree.depths.cpu().numpy()
    at = 0
    for p in split(parents, counts):
        assert np.array_equal(masks[at:at + len(p)], words_of(kin_of(p), words)) and depths[at:at + len(p)].tolist() == depths_of(p)
        at += len(p)


def test_trees_of_impossible_parents_and_of_too_many_nodes(ctx):
    """A parent that is no earlier node of the tree counts as none; a tree that does not fit is empty, its neighbours are not."""
    parents = [-1, 1, 0, 3, -7, 100, 2, 2 ** 31 - 1, -2 ** 31]
    sound = [-1, -1, 0, -1, -1, -1, 2, -1, -1]
    counts = [9, 33, 9]
    tree = K.DraftTree(ctx, pimdl, 51, most=32)
    tree.masks.fill_(-1)
    tree.build(ints(*parents, *range(-1, 32), *parents), starts_of(counts))
    torch.cuda.synchronize()
    want = words_of(kin_of(sound), 1)
    masks, depths = tree.masks.cpu().numpy(), tree.depths.cpu().numpy()
    for rows in (slice(0, 9), slice(42, 51)):
        assert np.array_equal(masks[rows], want) and depths[rows].tolist() == depths_of(sound)
    assert (masks[9:42] == 0).all() and (depths[9:42] == 0).all()


# ---------------------------------------------------------------------------------------------- attention

def reference_tree(q, k, v, parents, left, sinks, scale, gone=()):
    """q [n][heads][hd] of the tree's nodes, k and v [keys][kv_heads][hd], of which the last n are the tree's own: (out, how far fp32 may be off, sum p|v| / sum p).  gone: keys that are
    not there."""
    n, h, hd = q.shape
    keys, kv = k.shape[0], k.shape[1]
    old = keys - n
    depth = np.array(depths_of(parents))
    place = np.concatenate([np.arange(max(old, 0)), old + depth])
    seen = np.concatenate([np.ones((n, max(old, 0)), bool), kin_of(parents)], 1)
    if old < 0:  # nodes without a place are nobody's keys
        place, seen = place[-old:], seen[:, -old:]
    seen &= ((old + depth)[:, None] - place[None] <= left) | (place[None] < sinks)
    seen[:, list(gone)] = False
    seen = torch.from_numpy(seen).to(q.device)
    out, off, mass = (torch.zeros((n, h, hd), dtype=torch.float64, device=q.device) for _ in range(3))
    if keys == 0:
        return out, off, mass
    some = seen.any(-1, keepdim=True)
    for i in range(h):
        qh, kh, vh = q[:, i].double(), k[:, i // (h // kv)].double(), v[:, i // (h // kv)].double()
        s = torch.where(seen, (qh @ kh.t().contiguous()) * scale, -math.inf)
        ds = torch.where(seen, (hd + 8) * U * abs(scale) * (qh.abs() @ kh.abs().t().contiguous()), 0.0)
        p = torch.where(some, torch.softmax(s, -1), 0.0)
        out[:, i], mass[:, i] = p @ vh, p @ vh.abs()
        off[:, i] = (2 * torch.expm1(2 * ds.amax(-1, keepdim=True)) + 16 * U + 2 * (keys / 16 + 64) * U) * mass[:, i]
    return out, off, mass


def tree_case(ctx, seed, counts, lengths, heads, kv, hd, page_tokens, dtype, cache, left=None, sinks=0, width=None, scale=None, most=None, seen=check):
    f, n = Filled(ctx, seed, lengths, kv, hd, page_tokens, cache), sum(counts)
    parents = forest(counts, seed, width)
    tree = K.DraftTree(ctx, pimdl, n + 3, most=most or max(counts + [1]))
    tree.build(parents, starts_of(counts))
    wide = randn(gen_of(seed + 1), n + 2, heads * hd + 16, dtype=dtype)
    wide[n:] = float("nan")
    out = torch.full((n + 2, heads * hd), -5.0, device="cuda", dtype=TYPES[dtype])
    f.cache.attend(0, wide[:n, :heads * hd], out[:n], starts_of(counts), heads, left=left, sinks=sinks, scale=scale, tree=tree)
    torch.cuda.synchronize()
    assert (out[n:] == -5.0).all()
    at = 0
    for s, (c, p) in enumerate(zip(counts, split(parents, counts))):
        k, v = (x[0] for x in f.rows[s])
        if c:
            want, off, mass = reference_tree(wide[at:at + c, :heads * hd].reshape(c, heads, hd), k, v, p, 1 << 40 if left is None else left, sinks, 1 / math.sqrt(hd) if scale is None else scale)
            got = out[at:at + c].reshape(c, heads, hd)
            if seen is check:
                check(got, want, off, mass, dtype)
            else:
                check_pieces(got, want, off, mass, dtype, lengths[s], float(v.abs().max()))
        at += c
    return ctx.last_attention()


@pytest.mark.parametrize("dtype,cache", PAIRS)
@pytest.mark.parametrize("counts,lengths,heads,kv,hd,page_tokens,left,sinks,width", [
    ([1], [1], 1, 1, 64, 16, None, 0, None),                                       # the first token of all
    ([1, 1, 1], [777, 16, 17], 12, 12, 64, 16, None, 0, None),                     # trees of one node: single tokens
    ([24], [801], 12, 12, 64, 16, None, 0, 4),
    ([7, 1, 33], [40, 300, 33], 8, 1, 80, 16, None, 0, None),                      # a tree that is all there is
    ([64, 16, 0, 40], [700, 65, 9, 1000], 8, 2, 128, 32, None, 0, None),
    ([130, 2, 200], [1200, 70, 200], 4, 4, 96, 128, None, 0, 9),
    ([60, 33], [900, 500], 4, 2, 128, 16, 100, 4, None),                           # window and sinks
    ([60, 90], [600, 91], 6, 3, 32, 16, 2, 1, 2),                                  # windows that end within the branches
    ([60, 70], [60, 75], 4, 2, 64, 16, 3, 9, 1),                                   # ... and sinks that reach into them
    ([50, 20], [400, 30], 4, 2, 64, 32, 0, 0, None),                               # nothing but itself
    ([9, 3], [4, 0], 2, 2, 64, 16, None, 0, None),                                 # more nodes than keys: the first ones have no place
    ([5, 40], [70, 333], 2, 1, 24, 16, 20, 3, None),                               # the plain kernel
    ([60, 33, 1], [600, 33, 5], 6, 2, 72, 64, None, 0, 5),
    ([60, 30], [60, 50], 2, 2, 136, 16, 4, 2, 1),
    ([2, 20], [50, 61], 40, 1, 64, 16, None, 0, None),                             # 40 query heads to a key head
])
def test_trees_against_float64(ctx, dtype, cache, counts, lengths, heads, kv, hd, page_tokens, left, sinks, width):
    tree_case(ctx, sum(lengths) + hd, counts, lengths, heads, kv, hd, page_tokens, dtype, cache, left, sinks, width)


@pytest.mark.parametrize("old", [0, 1, 15, 16, 17, 31, 32, 33, 47, 48, 63, 64, 65])
@pytest.mark.parametrize("n", [1, 15, 31, 32, 33, 64, 65])
def test_trees_at_the_edges_of_tiles(ctx, old, n):
    """Where a tree begins and ends against tiles, pages and words of its masks."""
    tree_case(ctx, old + n, [n, n], [old + n, 2 * old + n], 4, 2, 64, 16, "f32", "f16")
    tree_case(ctx, old + n, [n], [old + n], 8, 2, 64, 16, "bf16", "bf16", left=7, sinks=2, width=2)


@pytest.mark.parametrize("dtype,cache,hd", [("bf16", "bf16", 128), ("f16", "f16", 64), ("f32", "f32", 64), ("f32", "f16", 80), ("f32", "bf16", 96)])
def test_large_trees_and_long_contexts(ctx, dtype, cache, hd):
    """Many rows, few rows over many keys, both in one batch, in splits; a tree of 1024 nodes."""
    tree_case(ctx, 1, [1024, 1, 300], [4000, 900, 301], 8, 2, hd, 16, dtype, cache)
    tree_case(ctx, 2, [33, 48], [20000, 30000], 8, 1, hd, 64, dtype, cache, width=8)
    tree_case(ctx, 3, [16], [9000], 2, 2, hd, 16, dtype, cache, left=5000, sinks=4)


# The plans that the sizes below have on 256 CUs; a rule that moves gets other sizes here, so that every way stays tested.
DEALT = dict(plain=0, wide=1, narrow=0, wide_splits=0, join=1)


def dealt(plan):
    assert {k: plan[k] for k in DEALT} == DEALT, plan


@pytest.mark.parametrize("n", [8, 9, 16, 17, 24, 31, 32, 33, 40, 41, 48, 49, 56, 64, 65, 80, 127, 128, 129, 192])
def test_dealt_blocks_of_any_number_of_rows(ctx, n):
    """1 to 8 groups of 32 rows, of which waves have whole tiles or halves, and several blocks; contexts that are cut over many shares, over few, and not at all."""
    dealt(tree_case(ctx, n, [n, 70, n, 40, n], [40000, 9000, n + 1, 300, n], 8, 2, 128, 64, "bf16", "bf16"))
    tree_case(ctx, n, [n, 3, n], [30000, 500, 8000 + n], 12, 3, 64, 16, "f32", "f16", left=9000, sinks=70, width=3)  # (fewer rows: blocks of 16)


@pytest.mark.parametrize("dtype,cache", PAIRS)
@pytest.mark.parametrize("hd", [32, 64, 80, 96, 128])
@pytest.mark.parametrize("left,sinks", [(None, 0), (4000, 4)])
def test_dealt_blocks_of_every_type_and_head_size(ctx, dtype, cache, hd, left, sinks):
    dealt(tree_case(ctx, hd, [100, 20, 33, 0, 150, 1], [9000, 900, 5033, 70, 150, 3000], 16, 8, hd, 16, dtype, cache, left, sinks))


def test_dealt_blocks_of_many_sequences(ctx):
    """As many as a deal takes, and one more, whose blocks are split evenly."""
    for batch in (512, 513):
        plan = tree_case(ctx, batch, [2, 5] * (batch // 2) + [3] * (batch % 2), [40, 90] * (batch // 2 - 1) + [40, 600] + [60] * (batch % 2), 48, 4, 32, 16, "bf16", "bf16")
        if batch == 512:
            dealt(plan)
        else:
            assert plan["wide"] and plan["narrow"] and plan["wide_splits"] >= 1, plan


def test_dealt_blocks_of_short_sequences(ctx):
    """More blocks than shares, which are not cut, and rows that see nothing."""
    dealt(tree_case(ctx, 7, [40, 64] * 30 + [1], [40, 100] * 30 + [3000], 8, 8, 64, 16, "f16", "f16"))
    dealt(tree_case(ctx, 8, [40, 64] * 30 + [1], [17, 0] * 30 + [3000], 8, 8, 64, 16, "f16", "f16"))


@pytest.mark.parametrize("batch,n,length,heads,kv,hd,dtype,cache,splits", [
    (4, 64, 1000, 32, 8, 128, "bf16", "bf16", 1),     # two blocks on every CU
    (2, 64, 4000, 32, 8, 128, "f16", "f16", 1),       # one, which is not split
    (4, 17, 7600, 32, 8, 128, "bf16", "bf16", 3),     # fewer, split up to two a CU
    (8, 60, 2000, 12, 12, 64, "f32", "f16", 1),
    (16, 24, 2000, 16, 16, 80, "f32", "f16", 1),      # 24 rows to a key head, which no other query head reads
    (16, 8, 4000, 32, 8, 64, "bf16", "bf16", 1),      # 32, of four heads of 64
    (8, 32, 4000, 16, 16, 128, "f32", "f32", 1),      # 32, of keys in fp32, where more are dealt out
    (3, 65, 1500, 8, 2, 96, "f32", "bf16", 3),        # 98 blocks, a CU each in thirds
])
def test_trees_in_blocks_of_sixteen_rows(ctx, batch, n, length, heads, kv, hd, dtype, cache, splits):
    """Trees whose scores are few enough for a CU, for the many blocks' sake, with lengths from the tree alone to all that the table holds."""
    lengths = [length if b == 0 else n + (length - n) * b // batch for b in range(batch)]
    plan = tree_case(ctx, n, [n - b % 2 for b in range(batch)], lengths, heads, kv, hd, 16, dtype, cache, width=5)
    want = dict(plain=0, wide=0, narrow=1, narrow_splits=splits, by_slot=1, join=int(splits > 1))
    assert {k: plan[k] for k in want} == want, plan


def test_dealt_blocks_recorded_and_replayed(ctx):
    """Lengths, borders of the batch, its list and its parents change from replay to replay, sequences that are not there among them; every replay against plain attention."""
    heads, kv, hd, room = 16, 8, 64, 340
    own, side = pimdl.Context(0), torch.cuda.Stream()
    f = Filled(own, 60, [9000, 5033, 900, 70], kv, hd, 16, "f16")
    full = f.cache.lengths.clone()
    tree, starts, seqs, parents = K.DraftTree(own, pimdl, room, most=160), starts_of([100, 150, 60, 30]), ints(0, 1, 2, 3), forest([100, 150, 60, 30], 1)
    q, out = randn(gen_of(61), room, heads * hd, dtype="f16"), torch.zeros(room, heads * hd, device="cuda", dtype=torch.float16)

    def step():
        tree.build(parents, starts)
        f.cache.attend(0, q, out, starts, heads, seqs, left=6000, sinks=70, tree=tree)

    torch.cuda.synchronize()
    own.set_stream(side.cuda_stream)
    with torch.cuda.stream(side):
        step()  # sizes the scratch
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side, capture_error_mode="thread_local"):
        step()
    dealt(own.last_attention())
    for i, (counts, lengths, order) in enumerate([([100, 150, 60, 30], [9000, 5033, 900, 70], [0, 1, 2, 3]), ([1, 160, 9, 33], [8000, 4000, 60, 33], [2, 0, 3, 1]),
                                                  ([0, 0, 150, 0], [9000, 5033, 900, 70], [0, 1, 2, 3]), ([33, 40, 50, 60], [40, 41, 50, 20], [3, 99, 0, -1]),
                                                  ([64, 64, 64, 64], [0, 3, 64, 70], [3, 2, 1, 0]), ([100, 150, 60, 30], [9000, 5033, 900, 70], [1, 0, 1, 2])]):
        torch.cuda.synchronize()
        f.cache.lengths.copy_(torch.minimum(ints(*lengths), full))
        starts.copy_(starts_of(counts))
        seqs.copy_(ints(*order))
        packed = forest(counts, 20 + i)
        parents.fill_(7)
        parents[:sum(counts)] = packed
        q.copy_(randn(gen_of(70 + i), *q.shape, dtype="f16"))
        out.fill_(-5.0)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert (out[sum(counts):] == -5.0).all(), i
        at = 0
        for c, s, p in zip(counts, order, split(packed, counts)):
            length = min(lengths[s], int(full[s])) if 0 <= s < 4 else 0
            k, v = (x[0][:length] for x in f.rows[s if 0 <= s < 4 else 0])
            if c:
                want, off, mass = reference_tree(q[at:at + c].reshape(c, heads, hd), k, v, p, 6000, 70, 1 / math.sqrt(hd))
                check(out[at:at + c].reshape(c, heads, hd), want, off, mass, "f16")
            at += c
    own.close()


@pytest.mark.parametrize("dtype,cache,hd", [("bf16", "bf16", 128), ("f16", "f16", 64), ("f32", "f32", 80), ("f32", "f16", 32), ("f32", "bf16", 96), ("f32", "f32", 64), ("f32", "bf16", 128)])
def test_dealt_blocks_over_pages_that_are_not_there(ctx, dtype, cache, hd):
    """... and past values that are not finite, which only those who see them get."""
    counts, lengths, heads, kv = [90, 130, 33], [9000, 4100, 700], 16, 8
    f, parents = Filled(ctx, 80, lengths, kv, hd, 16, cache), forest(counts, 81)
    gone = [[3, 4, 5, 6, 300, 8950 // 16], [0, 1, (4100 - 130 + 20) // 16], list(range(30))]
    for s, pages in enumerate(gone):
        for i, page in enumerate(pages):
            f.cache.tables[s, page] = (-1, 1 << 30, f.cache.k.shape[1])[i % 3]
    tree, n = K.DraftTree(ctx, pimdl, sum(counts), most=130), sum(counts)
    tree.build(parents, starts_of(counts))
    q = randn(gen_of(82), n, heads * hd, dtype=dtype)
    out = [torch.zeros_like(q) for _ in range(2)]
    f.cache.attend(0, q, out[0], starts_of(counts), heads, tree=tree)
    dealt(ctx.last_attention())
    at = 0
    for s, (c, p) in enumerate(zip(counts, split(parents, counts))):
        k, v = (x[0] for x in f.rows[s])
        want, off, mass = reference_tree(q[at:at + c].reshape(c, heads, hd), k, v, p, 1 << 40, 0, 1 / math.sqrt(hd), [j for j in range(lengths[s]) if j // 16 in gone[s]])
        check(out[0][at:at + c].reshape(c, heads, hd), want, off, mass, dtype)
        at += c
    # node 77 of the second tree: its own value is infinite, for one key head; its key is NaN, for another
    node, place = 77, 4100 - 130 + 77
    page = int(f.cache.tables[1, place // 16])
    f.cache.v[0, page, 2, place % 16, hd - 1] = float("inf")
    f.cache.k[0, page, 5, place % 16, 0] = float("nan")
    f.cache.attend(0, q, out[1], starts_of(counts), heads, tree=tree)
    torch.cuda.synchronize()
    of = [torch.from_numpy(kin_of(split(parents, counts)[1]))[:, node].nonzero()[:, 0].cuda() + 90, heads // kv]
    a, b = (o.reshape(n, heads, hd).clone() for o in out)
    assert not torch.isfinite(b[of[0], 2 * of[1]:3 * of[1], hd - 1]).any() and torch.isnan(b[of[0], 5 * of[1]:6 * of[1]]).all()
    for o in (a, b):
        o[of[0], 2 * of[1]:3 * of[1], hd - 1] = 0
        o[of[0], 5 * of[1]:6 * of[1]] = 0
    assert torch.equal(a, b)


def test_more_words_than_nodes_change_nothing(ctx):
    for most in (40, 64, 65, 1024):
        tree_case(ctx, 5, [40, 3], [200, 300], 4, 2, 64, 16, "bf16", "bf16", most=most)


@pytest.mark.parametrize("scale", [-0.2, 0.0, 3.0])
def test_scales_of_trees(ctx, scale):
    tree_case(ctx, 6, [40, 17], [200, 300], 4, 2, 64, 16, "f32", "f32", scale=scale)
    tree_case(ctx, 6, [40, 17], [200, 300], 4, 2, 72, 16, "f32", "f16", scale=scale)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("counts,lengths,hd", [([40, 64], [4000, 3000], 64), ([600, 1, 200], [3000, 900, 2000], 128), ([3, 5], [700, 900], 128)])
def test_trees_round_their_output_alone(ctx, dtype, counts, lengths, hd):
    tree_case(ctx, hd, counts, lengths, 8, 2, hd, 16, dtype, dtype, seen=check_pieces)


@pytest.mark.parametrize("dtype,cache", PAIRS)
@pytest.mark.parametrize("hd", [64, 72, 80, 128])
@pytest.mark.parametrize("left,sinks", [(None, 0), (50, 4)])
def test_a_chain_is_a_continuation(ctx, dtype, cache, hd, left, sinks):
    """Trees of one branch give what tokens that follow each other give, to the rounding of either."""
    counts, lengths = [40, 1, 7], [300, 77, 7]
    f, n = Filled(ctx, hd, lengths, 2, hd, 16, cache), sum(counts)
    q = randn(gen_of(hd), n, 8 * hd, dtype=dtype)
    plain, treed = torch.zeros_like(q), torch.zeros_like(q)
    tree = K.DraftTree(ctx, pimdl, n)
    tree.build(ints(*[i - 1 for c in counts for i in range(c)]), starts_of(counts))
    f.cache.attend(0, q, plain, starts_of(counts), 8, left=left, sinks=sinks)
    f.cache.attend(0, q, treed, starts_of(counts), 8, left=left, sinks=sinks, tree=tree)
    torch.cuda.synchronize()
    at = 0
    for s, c in enumerate(counts):
        k, v = (x[0] for x in f.rows[s])
        want, off, mass = reference_tree(q[at:at + c].reshape(c, 8, hd), k, v, list(range(-1, c - 1)), 1 << 40 if left is None else left, sinks, 1 / math.sqrt(hd))
        for out in (plain, treed):
            check(out[at:at + c].reshape(c, 8, hd), want, off, mass, dtype)
        at += c


@pytest.mark.parametrize("dtype,cache", PAIRS)
@pytest.mark.parametrize("hd,nodes", [(64, 40), (64, 300), (80, 40), (24, 40), (128, 1000)])
def test_what_a_tree_hides_changes_nothing(ctx, dtype, cache, hd, nodes):
    """Infinities and NaN in the keys and values of a node reach its descendants and itself, and nobody else bit for bit; what lies behind a sequence reaches nobody."""
    lengths, heads = [100 + nodes], 4
    f, p = Filled(ctx, 1, lengths, 2, hd, 16, cache), forest([nodes], 4)
    tree, at = K.DraftTree(ctx, pimdl, nodes, most=nodes), starts_of([nodes])
    tree.build(p, at)
    q = randn(gen_of(2), nodes, heads * hd, dtype=dtype)
    kin = torch.from_numpy(kin_of(p.tolist())).cuda()

    def run():
        out = torch.zeros_like(q)
        f.cache.attend(0, q, out, at, heads, tree=tree)
        torch.cuda.synchronize()
        return out

    plain = run()
    assert torch.isfinite(plain).all()
    node = 2
    page, row = int(f.cache.tables[0, (100 + node) // 16]), (100 + node) % 16
    for pool in (f.cache.k, f.cache.v):
        keep = pool[0, page, :, row].clone()
        for bad in (float("inf"), float("-inf"), float("nan")):
            pool[0, page, :, row, 3] = bad
            got = run()
            others = ~kin[:, node]
            assert torch.equal(got[others], plain[others])
            hit = got[kin[:, node]].reshape(-1, heads, hd)
            if pool is f.cache.v:
                assert not torch.isfinite(hit[..., 3]).any() and torch.isfinite(hit[..., 4:]).all()
            elif bad != bad:
                assert not torch.isfinite(hit).any()
            pool[0, page, :, row] = keep
    assert torch.equal(run(), plain)


@pytest.mark.parametrize("dtype,cache", PAIRS)
@pytest.mark.parametrize("hd,nodes,heads", [(64, 40, 2), (64, 400, 8), (24, 40, 2)])
def test_trees_over_pages_that_are_not_there(ctx, dtype, cache, hd, nodes, heads):
    old = 150
    f, p = Filled(ctx, 12, [old + nodes], 2, hd, 16, cache), forest([nodes], 3)
    gone = [1, 4, (old + 20) // 16]
    for page, entry in zip(gone, (-1, 1 << 30, f.cache.k.shape[1])):
        f.cache.tables[0, page] = entry
    tree, at = K.DraftTree(ctx, pimdl, nodes, most=nodes), starts_of([nodes])
    tree.build(p, at)
    q = randn(gen_of(13), nodes, heads * hd, dtype=dtype)
    out = torch.zeros_like(q)
    f.cache.attend(0, q, out, at, heads, tree=tree)
    torch.cuda.synchronize()
    k, v = (x[0] for x in f.rows[0])
    want, off, mass = reference_tree(q.reshape(nodes, heads, hd), k, v, p.tolist(), 1 << 40, 0, 1 / math.sqrt(hd), [j for j in range(old + nodes) if j // 16 in gone])
    check(out.reshape(nodes, heads, hd), want, off, mass, dtype)


def test_trees_without_masks_see_the_context(ctx):
    """A tree of more nodes than there are bits: its tokens see what the cache held before, and nothing where it held nothing."""
    f, heads = Filled(ctx, 3, [100, 40, 50], 2, 64, 16, "f16"), 4
    counts = [40, 40, 9]
    tree, q = K.DraftTree(ctx, pimdl, 89, most=32), randn(gen_of(1), 89, heads * 64)
    tree.build(forest(counts, 1), starts_of(counts))
    out = torch.zeros_like(q)
    f.cache.attend(0, q, out, starts_of(counts), heads, tree=tree)
    torch.cuda.synchronize()
    k, v = (x[0] for x in f.rows[0])
    want, off, mass = reference_tree(q[:40].reshape(40, heads, 64), k, v, [-1] * 40, 1 << 40, 0, 0.125, range(60, 100))
    check(out[:40].reshape(40, heads, 64), want, off, mass, "f32")
    assert (out[40:80] == 0).all()


# ---------------------------------------------------------------------------------------------- accept

class Book:
    """What accepting does, as a sequential program does it."""

    def __init__(self, cache):
        self.tables, self.lengths, self.refs = (t.cpu().numpy().astype(np.int64) for t in (cache.tables, cache.lengths, cache.refs))
        self.k, self.v = cache.k.cpu().clone(), cache.v.cpu().clone()
        self.pt, self.lacking = cache.page_tokens, int(cache.lacking)

    def accept(self, counts, seqs, parents, last):
        kept, done, refs = [], set(), self.refs.copy()
        for b, (n, s, p, end) in enumerate(zip(counts, seqs, parents, last)):
            kept.append(-1)
            first = s not in done
            done.add(s)
            if not first or self.lacking or not 0 <= s < len(self.lengths) or not -1 <= end < n or n > self.lengths[s]:
                continue
            path, at = [], end
            while at >= 0:
                path.insert(0, at)
                at = p[at]
            base = int(self.lengths[s]) - n
            moved = next((j for j, i in enumerate(path) if i != j), len(path))
            used = self.tables[s, (base + moved) // self.pt:-(-(base + len(path)) // self.pt)]
            if n and any(0 <= g < len(refs) and refs[g] > 1 for g in used):
                continue
            kept[-1] = len(path)
            where = lambda j: (int(self.tables[s, j // self.pt]), j % self.pt)  # noqa: E731
            there = lambda g: 0 <= g < len(refs)  # noqa: E731
            for pool in (self.k, self.v):
                old = pool.clone()
                for j, i in enumerate(path):
                    (f, fr), (t, tr) = where(base + i), where(base + j)
                    if there(f) and there(t):
                        pool[:, t, :, tr] = old[:, f, :, fr]
            for j in range(-(-(base + len(path)) // self.pt), -(-int(self.lengths[s]) // self.pt)):
                if there(self.tables[s, j]):
                    self.refs[self.tables[s, j]] -= 1
                self.tables[s, j] = -1
            self.lengths[s] = base + len(path)
        return kept

    def same(self, cache):
        for mine, theirs in ((self.tables, cache.tables), (self.lengths, cache.lengths), (self.refs, cache.refs)):
            assert np.array_equal(mine, theirs.cpu().numpy())
        bits = torch.int32 if cache.k.dtype == torch.float32 else torch.int16
        for mine, theirs in ((self.k, cache.k), (self.v, cache.v)):
            assert torch.equal(mine.view(bits), theirs.cpu().view(bits))


def accept_case(ctx, cache, counts, seqs, parents, last, most=None, given=None):
    at, n = starts_of(counts), sum(counts)
    tree = K.DraftTree(ctx, pimdl, n, most=most or max(counts + [1]))
    tree.build(parents, at)
    book, kept = Book(cache), torch.full((len(counts),), -9, device="cuda", dtype=torch.int32)
    want = book.accept(counts, list(range(len(counts))) if seqs is None else seqs, split(parents, counts) if given is None else given, last)
    cache.accept(tree, ints(*last), kept, at, None if seqs is None else ints(*seqs))
    torch.cuda.synchronize()
    assert kept.tolist() == want
    book.same(cache)
    return want


@pytest.mark.parametrize("cache,kv,hd", [("f32", 2, 64), ("f16", 3, 80), ("bf16", 1, 31), ("bf16", 2, 17), ("f32", 1, 1), ("f16", 1, 1), ("bf16", 8, 128), ("f16", 5, 2)])
@pytest.mark.parametrize("page_tokens", [16, 64])
def test_accept_against_a_sequential_model(ctx, cache, kv, hd, page_tokens):
    """Branches of any length, whole trees, none; parts of pages and whole ones given back; rows of any size."""
    lengths = [100, 64, 40, 33, 200, 16, 48, 70, 90]
    counts = [40, 64, 8, 1, 100, 0, 16, 33, 90]
    parents = torch.cat([forest(counts[:4], 3), forest([100], 0, width=1), forest(counts[6:8], 5), forest([90], 0, width=4)])
    for rnd in range(3):
        g = Filled(ctx, hd, lengths, kv, hd, page_tokens, cache, layers=3)
        last = [[39, 63, 7, 0, 99, -1, 15, 32, 89], [-1, 0, -1, -1, 50, -1, 3, 20, 17], [17, 40, 3, 0, 98, -1, -1, 1, 50]][rnd]
        accept_case(ctx, g.cache, counts, None, parents, last)


def test_accept_of_large_trees(ctx):
    """Up to 1024 nodes: branches of all of them, of every second, of few."""
    for width, last in ((1, 1023), (2, 1022), (7, 1000), (None, 1023)):
        f = Filled(ctx, 2, [1100, 1024], 2, 64, 32, "bf16", layers=2)
        accept_case(ctx, f.cache, [1024, 1024], None, forest([1024, 1024], 9, width), [last, last - 3])


def test_accept_leaves_what_it_cannot_do(ctx):
    """Nodes that are not there, sequences that are not there or listed twice, more nodes than positions, trees without masks."""
    f = Filled(ctx, 4, [100, 64, 40, 33, 20], 2, 64, 16, "f16", layers=2)
    counts, seqs = [10, 10, 10, 10, 25, 10], [0, 7, 2, 0, 4, -1]
    p = forest(counts, 2)
    assert accept_case(ctx, f.cache, counts, seqs, p, [5, 5, 10, 5, 5, 5])[1:] == [-1] * 5
    assert accept_case(ctx, f.cache, [10, 10], [1, 3], forest([10, 10], 2), [-2, 2 ** 31 - 1]) == [-1, -1]
    # 40 nodes in masks of 32: no tree; a mask without its own node: the same
    tree, kept = K.DraftTree(ctx, pimdl, 40, most=32), ints(5)
    tree.build(forest([40], 1), starts_of([40]))
    book = Book(f.cache)
    f.cache.accept(tree, ints(3), kept, starts_of([40]), ints(1))
    torch.cuda.synchronize()
    assert kept.tolist() == [-1]
    f.cache.accept(tree, ints(3), kept, starts_of([10]), ints(1))
    torch.cuda.synchronize()
    assert kept.tolist() == [-1]
    book.same(f.cache)


def test_accept_while_pages_were_lacking(ctx):
    """The tree is not in the cache then: the newest positions are older tokens."""
    cache = small_cache(ctx, 5, pages=3, seqs=2, width=8)
    cache.reserve(ints(0), ints(40))
    cache.reserve(ints(0), ints(20))
    assert int(cache.lacking) == 1
    assert accept_case(ctx, cache, [20], [0], forest([20], 1), [5]) == [-1]
    cache.reserve(ints(0), ints(8))
    assert accept_case(ctx, cache, [8], [0], forest([8], 1), [-1]) == [0]


def test_accept_does_not_write_on_pages_of_others(ctx):
    """A fork made while the draft was there holds its whole pages too: a sequence that would write on them, or leave one partly filled, is left; one whose pages stay as they are, or
    go, is not."""
    cache = small_cache(ctx, 6, pages=60, seqs=9, width=8)
    cache.reserve(ints(0, 1, 2, 3), ints(80, 80, 80, 70))
    cache.fork(ints(0, 1, 2), ints(4, 5, 6))
    counts = [48, 48, 48, 40]
    p = torch.cat([forest([48], 0, width=1), forest([48], 0, width=2), forest([48], 0, width=1), forest([40], 0, width=3)])
    # 0: all of a chain, nothing changes; 1: rows would move; 2: a page would be left partly filled; 3: nobody else's
    assert accept_case(ctx, cache, counts, [0, 1, 2, 3], p, [47, 40, 20, 30]) == [48, -1, -1, 11]
    # whole pages go, what stays is full: 80 - 48 = 32 positions
    assert accept_case(ctx, cache, [48], [1], forest([48], 1), [-1]) == [0]
    cache.free(ints(6))
    assert accept_case(ctx, cache, [48], [2], forest([48], 0, width=1), [20]) == [21]


def test_accept_finds_a_page_of_others_wherever_it_lies(ctx):
    """A page that another sequence holds, the first, a middle or the last one of 65 that rows would move to, each looked at by a thread of its own: the sequence is left
    as it was, the one beside it is not."""
    p = torch.cat([ints(-1, -1, *range(1, 1023)), forest([1024], 3, width=5)])
    for place in (4, 35, 67, 68):
        f = Filled(ctx, 8, [1100, 1100], 2, 64, 16, "bf16", layers=9)
        f.cache.refs[f.cache.tables[0, place].long()] += 1
        assert accept_case(ctx, f.cache, [1024, 1024], None, p, [1023, 1000])[0] == -1
    f = Filled(ctx, 8, [1100, 1100], 2, 64, 16, "bf16", layers=9)
    f.cache.refs[f.cache.tables[0, 3].long()] += 1  # (before all of them)
    assert accept_case(ctx, f.cache, [1024, 1024], None, p, [1023, 1000])[0] == 1023


def test_accept_of_pages_that_are_not_there(ctx):
    f = Filled(ctx, 4, [100, 64], 2, 64, 16, "f16", layers=2)
    f.cache.tables[0, 5], f.cache.tables[1, 0] = -1, 1 << 28
    accept_case(ctx, f.cache, [60, 64], None, forest([60, 64], 0, width=3), [57, 60])


# ---------------------------------------------------------------------------------------------- together

@pytest.mark.parametrize("dtype,hd", [("f32", 64), ("bf16", 128), ("f16", 72)])
def test_drafts_go_on_from_what_was_accepted(ctx, dtype, hd):
    """Prompts, drafts and accepted branches of three sequences, with a fork, a freed sequence and a compaction between: what each node is given lies in the cache turned by its
    position, and its attention is float64's over its own branch."""
    heads, kv, layers, pairs = 4, 2, 2, "halves"
    cache, r = K.PagedCache(ctx, pimdl, layers, 200, kv, hd, 16, "f32" if dtype == "f32" else dtype, 5, 600), rotary_of(ctx, hd, hd, pairs)
    given = {s: [([], []) for _ in range(layers)] for s in range(5)}  # keys and values as the cache has them
    gen, rng = gen_of(31), np.random.default_rng(31)

    def step(seqs, counts, chain):
        lst, n, starts = ints(*seqs), sum(counts), starts_of(counts)
        parents = ints(*[i - 1 for c in counts for i in range(c)]) if chain else forest(counts, int(rng.integers(1 << 30)))
        branches = split(parents, counts)
        cache.reserve(lst, ints(*counts))
        tree = K.DraftTree(ctx, pimdl, n, most=max(counts))
        tree.build(parents, starts)
        last = [c - 1 if chain else int(rng.integers(-1, c)) for c in counts]
        kept = torch.zeros(len(seqs), device="cuda", dtype=torch.int32)
        base = [sum(x.shape[0] for x in given[s][0][0]) for s in seqs]
        place = torch.tensor(np.concatenate([b + np.array(depths_of(p)) for b, p in zip(base, branches)]), device="cuda")
        for layer in range(layers):
            x = randn(gen, n, (heads + 2 * kv) * hd, dtype=dtype)
            q, k, v = x[:, :heads * hd], x[:, heads * hd:(heads + kv) * hd], x[:, (heads + kv) * hd:]
            raw, out = q.clone(), torch.zeros(n, heads * hd, device="cuda", dtype=TYPES[dtype])
            cache.append(layer, k, v, starts, lst, rotary=r, q=q, q_out=q, tree=tree)
            cache.attend(layer, q, out, starts, heads, lst, tree=tree)
            torch.cuda.synchronize()
            want, off = turned(raw, place, r.freqs, pairs, hd)
            check_turned(q, want, off, dtype)
            want_k, off_k = turned(k, place, r.freqs, pairs, hd)
            at = 0
            for s, c, b, p, end in zip(seqs, counts, base, branches, last):
                slots = torch.arange(b, b + c, device="cuda")
                pages = cache.tables[s].long()[slots // 16]
                kk, vv = cache.k[layer, pages, :, slots % 16], cache.v[layer, pages, :, slots % 16]
                check_turned(kk.flatten(1), want_k[at:at + c], off_k[at:at + c], dtype)
                assert torch.equal(vv.flatten(1), v[at:at + c])
                ks, vs = (torch.cat(old + [new]) for old, new in zip(given[s][layer], (kk, vv)))
                want, o, mass = reference_tree(q[at:at + c].reshape(c, heads, hd), ks, vs, p, 1 << 40, 0, 1 / math.sqrt(hd))
                check(out[at:at + c].reshape(c, heads, hd), want, o, mass, dtype)
                path = [i for i in range(end + 1) if kin_of(p)[end, i]]
                given[s][layer][0].append(kk[path])
                given[s][layer][1].append(vv[path])
                at += c
        cache.accept(tree, ints(*last), kept, starts, lst)
        torch.cuda.synchronize()
        for s, got in zip(seqs, kept.tolist()):
            assert got == given[s][0][0][-1].shape[0] and int(cache.lengths[s]) == sum(x.shape[0] for x in given[s][0][0])

    step([0, 3], [70, 7], True)
    step([0, 3], [20, 33], False)
    cache.fork(ints(0), ints(1))
    given[1] = [tuple(list(x) for x in pair) for pair in given[0]]
    step([1, 0, 3], [40, 1, 9], False)
    cache.free(ints(0))
    given[0] = [([], []) for _ in range(layers)]
    cache.compact()
    step([3, 1], [17, 50], False)
    step([0, 1, 3], [30, 1, 1], True)
    step([0, 1, 3], [30, 8, 16], False)
    held = sum(-(-int(n) // 16) for n in cache.lengths)
    assert int((cache.refs > 0).sum()) == held  # nothing shared any more, nothing lost


def test_a_captured_step_follows_trees_and_branches(ctx):
    """A whole step (room, tree, append, attention, accept) recorded into a graph: every replay, with parents and branches of its own, against the eager calls, other work between them."""
    heads, kv, hd, counts = 8, 2, 64, [24, 40, 1]
    own, side, n = pimdl.Context(0), torch.cuda.Stream(), sum(counts)
    made = []
    for c in (ctx, own):
        cache = K.PagedCache(c, pimdl, 2, 400, kv, hd, 16, "bf16", 3, 2000)
        cache.reserve(ints(0, 1, 2), ints(500, 30, 1290))
        for pool, seed in ((cache.k, 1), (cache.v, 2)):
            pool.copy_(randn(gen_of(seed), *pool.shape, dtype="bf16"))
        made.append((cache, rotary_of(c, hd, hd, "neighbours"), K.DraftTree(c, pimdl, n, most=40), torch.zeros(n, heads * hd, device="cuda", dtype=torch.bfloat16), ints(0, 0, 0)))
        torch.cuda.synchronize()
        own.synchronize()
    seqs, news, starts, last = ints(0, 1, 2), ints(*counts), starts_of(counts), ints(3, 7, 0)
    parents, x = forest(counts, 1), randn(gen_of(3), n, (heads + 2 * kv) * hd, dtype="bf16")
    turns = [torch.zeros(n, heads * hd, device="cuda", dtype=torch.bfloat16) for _ in range(2)]

    def step(which):
        cache, r, tree, out, kept = made[which]
        cache.reserve(seqs, news)
        tree.build(parents, starts)
        for layer in range(2):
            cache.append(layer, x[:, heads * hd:(heads + kv) * hd], x[:, (heads + kv) * hd:], starts, seqs, rotary=r, q=x[:, :heads * hd], q_out=turns[which], tree=tree)
            cache.attend(layer, turns[which], out, starts, heads, seqs, tree=tree)
        cache.accept(tree, last, kept, starts, seqs)

    torch.cuda.synchronize()
    own.set_stream(side.cuda_stream)
    with torch.cuda.stream(side):
        step(1)  # sizes the scratch
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side, capture_error_mode="thread_local"):
        step(1)
    step(0)
    rng = np.random.default_rng(5)
    for i in range(6):
        torch.cuda.synchronize()
        parents.copy_(forest(counts, 10 + i))
        last.copy_(ints(*[int(rng.integers(-1, c)) for c in counts]))
        x.copy_(randn(gen_of(10 + i), *x.shape, dtype="bf16"))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        step(0)
        torch.cuda.synchronize()
        a, b = made
        assert torch.equal(a[3], b[3]) and torch.equal(turns[0], turns[1]) and a[4].tolist() == b[4].tolist() and min(a[4].tolist()) >= 0, i
        for one, two in ((a[0].lengths, b[0].lengths), (a[0].tables, b[0].tables), (a[0].refs, b[0].refs), (a[0].k, b[0].k), (a[0].v, b[0].v), (a[2].masks, b[2].masks)):
            assert torch.equal(one, two), i
    own.close()


def test_two_contexts_draft_on_two_streams(ctx):
    """Two caches, each with its own context and stream, at the same time."""
    jobs = []
    for i in range(2):
        c, st = pimdl.Context(0), torch.cuda.Stream()
        c.set_stream(st.cuda_stream)
        f, p = Filled(c, 30 + i, [3000 + 500 * i, 60], 2, 64, 16, "f16"), forest([30, 41], i)
        tree, q = K.DraftTree(c, pimdl, 71, most=64), randn(gen_of(40 + i), 71, 8 * 64)
        jobs.append((c, f, p, tree, q, torch.zeros_like(q), starts_of([30, 41])))
    torch.cuda.synchronize()
    for _ in range(20):
        for c, f, p, tree, q, out, starts in jobs:
            tree.build(p, starts)
            f.cache.attend(0, q, out, starts, 8, tree=tree)
    torch.cuda.synchronize()
    for i, (c, f, p, tree, q, out, starts) in enumerate(jobs):
        at = 0
        for s, (n, b) in enumerate(zip([30, 41], split(p, [30, 41]))):
            k, v = (x[0] for x in f.rows[s])
            want, off, mass = reference_tree(q[at:at + n].reshape(n, 8, 64), k, v, b, 1 << 40, 0, 0.125)
            check(out[at:at + n].reshape(n, 8, 64), want, off, mass, "f32")
            at += n
        c.close()


def test_a_tree_of_another_context(ctx):
    """Filled by one context and read by another, each on a stream of its own, with another forest every time; contexts on given streams that differ are refused."""
    one, two = pimdl.Context(0), pimdl.Context(0)
    f, counts = Filled(two, 33, [3000, 1100], 2, 64, 16, "f16"), [60, 1000]
    tree, q, starts = K.DraftTree(one, pimdl, 1060, most=1024), randn(gen_of(7), 1060, 8 * 64), starts_of(counts)
    forests, outs = [forest(counts, i, width=1 + 3 * i) for i in range(6)], [torch.zeros_like(q) for _ in range(6)]
    torch.cuda.synchronize()
    for p, out in zip(forests, outs):
        tree.build(p, starts)
        f.cache.attend(0, q, out, starts, 8, tree=tree)
    torch.cuda.synchronize()
    mine = K.DraftTree(two, pimdl, 1060, most=1024)
    for p, out in zip(forests, outs):
        mine.build(p, starts)
        again = torch.zeros_like(q)
        torch.cuda.synchronize()
        f.cache.attend(0, q, again, starts, 8, tree=mine)
        torch.cuda.synchronize()
        assert torch.equal(out, again)
    two.set_stream(torch.cuda.Stream().cuda_stream)
    with pytest.raises(ValueError, match="another stream"):
        f.cache.attend(0, q, outs[0], starts, 8, tree=tree)
    two.close()
    tree.build(forests[0], starts)  # (a reader that is gone)
    torch.cuda.synchronize()
    one.close()


def test_drafts_beyond_four_gigabytes(ctx):
    """Pages whose offsets do not fit in 32 bits, of bytes or of elements: written turned, attended to, moved."""
    kv, hd, pt, pages = 2, 128, 16, 700_000  # 8 KiB a page of 16 bits: 5.7 GB
    k, v = (torch.zeros(1, pages, kv, pt, hd, device="cuda", dtype=torch.float16) for _ in range(2))
    tables, refs = torch.full((1, 8), -1, device="cuda", dtype=torch.int32), torch.zeros(pages, device="cuda", dtype=torch.int32)
    mine = [5, pages - 1, 600_000, pages - 70]
    tables[0, :4] = ints(*mine)
    refs[mine] = 1
    cache, r = K.PagedCache.over(ctx, pimdl, k, v, tables, ints(60), refs), rotary_of(ctx, hd, hd, "halves")
    for pool in (k, v):
        pool[0, mine] = randn(gen_of(1), 4, kv, pt, hd, dtype="f16")
    n, heads, p = 40, 4, forest([40], 0, width=3)
    tree, starts = K.DraftTree(ctx, pimdl, n), starts_of([n])
    tree.build(p, starts)
    x = randn(gen_of(2), n, (heads + 2 * kv) * hd, dtype="f16")
    out = torch.zeros(n, heads * hd, device="cuda", dtype=torch.float16)
    cache.append(0, x[:, heads * hd:(heads + kv) * hd], x[:, (heads + kv) * hd:], starts, rotary=r, q=x[:, :heads * hd], q_out=x[:, :heads * hd], tree=tree)
    cache.attend(0, x[:, :heads * hd], out, starts, heads, tree=tree)
    torch.cuda.synchronize()
    rows = [(mine[j // 16], j % 16) for j in range(60)]
    kk, vv = (torch.stack([pool[0, a, :, b] for a, b in rows]) for pool in (k, v))
    place = 20 + torch.tensor(depths_of(p.tolist()), device="cuda")
    want, off = turned(x[:, heads * hd:(heads + kv) * hd], place, r.freqs, "halves", hd)
    check_turned(kk[20:].flatten(1), want, off, "f16")
    assert torch.equal(vv[20:].flatten(1), x[:, (heads + kv) * hd:])
    want, off, mass = reference_tree(x[:, :heads * hd].reshape(n, heads, hd), kk, vv, p.tolist(), 1 << 40, 0, 1 / math.sqrt(hd))
    check(out.reshape(n, heads, hd), want, off, mass, "f16")
    kept = ints(0)
    cache.accept(tree, ints(37), kept, starts)
    torch.cuda.synchronize()
    path = [i for i in range(38) if kin_of(p.tolist())[37, i]]
    assert kept.tolist() == [len(path)] and int(cache.lengths[0]) == 20 + len(path)
    for j, i in enumerate(path):
        a, b = rows[20 + j]
        assert torch.equal(k[0, a, :, b], kk[20 + i]) and torch.equal(v[0, a, :, b], vv[20 + i])
    assert cache.tables[0].tolist() == [m if i * 16 < 20 + len(path) else -1 for i, m in enumerate(mine)] + [-1] * 4


# ---------------------------------------------------------------------------------------------- refusals

def test_wrong_calls_are_refused(ctx):
    f, r = Filled(ctx, 50, [40, 9], 2, 64, 16, "f16"), rotary_of(ctx, 64, 64, "halves")
    c, x, q = f.cache, randn(gen_of(1), 2, 128), randn(gen_of(2), 3, 256)[:2]
    before = (c.k.clone(), c.tables.clone())
    tree = K.DraftTree(ctx, pimdl, 2)
    calls = [
        lambda: r.rotate(q, x, q.as_strided((2, 256), (300, 1)), x, starts_of([1, 1])),           # in place with another stride
        lambda: c.append(0, x.bfloat16(), x.bfloat16(), starts_of([1, 1]), rotary=r),             # of another type than the cache
        lambda: c.append(0, x, x, starts_of([1, 1, 0]), rotary=r),                                # more rows than sequences
        lambda: c.attend(0, q, torch.zeros_like(q), starts_of([1, 1, 0]), 4, tree=tree),
        lambda: c.attend(0, q, torch.zeros_like(q), starts_of([1, 1]), 3, tree=tree),             # heads that do not share evenly
        lambda: c.append(0, x, x, starts_of([1, 1]).cpu(), rotary=r),                             # host memory
        lambda: tree.build(ints(-1, -1).cpu(), starts_of([1, 1])),
        lambda: c.accept(tree, ints(0, 0).cpu(), ints(0, 0), starts_of([1, 1])),
    ]
    for call in calls:
        with pytest.raises((ValueError, pimdl.PimdlError)):
            call()
    torch.cuda.synchronize()
    assert torch.equal(c.k.view(torch.int16), before[0].view(torch.int16)) and torch.equal(c.tables, before[1])


def test_accept_refuses_to_write_over_what_it_reads(ctx):
    f, tree = Filled(ctx, 50, [40, 9], 2, 64, 16, "f16"), K.DraftTree(ctx, pimdl, 2)
    before, both = f.cache.lengths.clone(), ints(-1, -1, 0, 1, 2)
    last, mixed, starts, seqs = both[:2], both[1:3], starts_of([1, 1]), ints(0, 1)
    for args in ((last, last, starts), (last, mixed, starts), (mixed, last, starts), (last, starts[:2], starts), (last, starts[1:], starts), (last, seqs, starts, seqs)):
        with pytest.raises(pimdl.PimdlError, match="overlap"):
            f.cache.accept(tree, *args)
    torch.cuda.synchronize()
    assert torch.equal(f.cache.lengths, before)
    f.cache.accept(tree, last, both[2:4], starts)  # beside each other


def test_calls_without_tokens_do_nothing(ctx):
    f, r = Filled(ctx, 50, [40, 9], 2, 64, 16, "f16"), rotary_of(ctx, 64, 64, "halves")
    book, tree, kept = Book(f.cache), K.DraftTree(ctx, pimdl, 0), ints(7, 7)
    x, none = torch.zeros(0, 128, device="cuda"), starts_of([0, 0])
    r.rotate(x, x, x, x, none)
    tree.build(ints(), none)
    f.cache.append(0, x, x, none, rotary=r, q=x, q_out=x, tree=tree)
    f.cache.attend(0, x, x, none, 2, tree=tree)
    torch.cuda.synchronize()
    book.same(f.cache)
    tree = K.DraftTree(ctx, pimdl, 4)  # (a tree's tensors that hold something)
    f.cache.accept(tree, ints(-1, -1), kept, none)
    torch.cuda.synchronize()
    assert kept.tolist() == [0, 0]
    book.same(f.cache)


def test_accept_of_a_tree_without_tokens(ctx):
    """As for a tree with room whose rows are empty: nothing moves, 0 are kept, and a row that cannot be done is still told."""
    f, none, kept = Filled(ctx, 50, [40, 9], 2, 64, 16, "f16"), starts_of([0, 0]), ints(7, 7)
    book = Book(f.cache)
    for tree in (K.DraftTree(ctx, pimdl, 0), K.DraftTree(ctx, pimdl, 0, most=1024)):
        for last, seqs, want in (((-1, -1), None, [0, 0]), ((-1, -1), (1, 1), [0, -1]), ((-1, 0), (0, 1), [0, -1]), ((-1, -1), (0, 2), [0, -1])):
            f.cache.accept(tree, ints(*last), kept, none, None if seqs is None else ints(*seqs))
            torch.cuda.synchronize()
            assert kept.tolist() == want
            book.same(f.cache)


# ---------------------------------------------------------------------------------------------- the transformer

def rotated_model(ctx, hd, heads, layers, seq_len, batch, rotary, window=None, fused=False):
    model, p = unrotated_model(ctx, hd, heads, layers, seq_len, batch, window, fused)
    p.rotary = rotary
    for layer in model.layers:
        layer.rotary = K.Rotary(ctx, pimdl, hd, **p.turns())
    return model, p


@pytest.mark.parametrize("hd,heads,window,fused", [(64, 4, None, False), (64, 4, (20, 5, 1), True), (24, 4, None, False)])
def test_layer_with_a_rotation(ctx, hd, heads, window, fused):
    """Whole sequences: q and k of the layer turned by their places, attention over what came out; eager and recorded."""
    plain, _ = unrotated_model(ctx, hd, heads, 1, 70, 3, window, fused)
    model, p = rotated_model(ctx, hd, heads, 1, 70, 3, (10000.0, hd // 2, "neighbours"), window, fused)
    x, raw, keep = randn(gen_of(1), p.n, p.token_dim), {}, {}
    plain.layers[0].forward(x, raw)
    model.layers[0].forward(x, keep)
    torch.cuda.synchronize()
    r = model.layers[0].rotary
    for name in "qk":
        want, off = turned(raw[name], places_of([70] * 3), r.freqs, "neighbours", hd)
        check_turned(keep[name], want, off, "f32")
    assert torch.equal(raw["v"], keep["v"])
    left, right, sinks = (1 << 40, 1 << 40, 0) if window is None else window
    j = torch.arange(70, device="cuda")
    seen = (j[None] <= j[:, None] + right) & ((j[None] + left >= j[:, None]) | (j[None] < sinks))
    for b in range(3):
        rows = slice(70 * b, 70 * b + 70)
        q, k, v = (keep[m][rows].reshape(70, heads, hd).double() for m in "qkv")
        for h in range(heads):
            s = (q[:, h] @ k[:, h].t().contiguous()) / math.sqrt(hd)
            ds = (hd + 8) * U / math.sqrt(hd) * (q[:, h].abs() @ k[:, h].abs().t().contiguous())
            share = torch.softmax(s.masked_fill(~seen, -math.inf), -1)
            mass = share @ v[:, h].abs()
            off = (2 * torch.expm1(2 * ds.amax(-1, keepdim=True)) + 16 * U + 2 * (70 / 16 + 64) * U) * mass
            check(keep["attn"][rows, h * hd:(h + 1) * hd], share @ v[:, h], off, mass, "f32")
    graph, static_x, static_y = model.capture(x)
    for i in range(3):
        static_x.copy_(x * (i + 1))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(static_y, model.forward(static_x))
    plain.close()
    model.close()


def test_a_model_built_with_a_rotation_has_it(ctx):
    from pim_dl_asplos_amd import transformer as T
    plain, p = unrotated_model(ctx, 64, 4, 1, 16, 1)
    p.rotary = (500000.0, None, "halves")
    layer = T.TransformerLayer(ctx, pimdl, T.synth_layers(p, ctx, pimdl, seed=3)[0], p)
    assert layer.rotary.dims == 64 and layer.rotary.pairs == "halves" and abs(float(layer.rotary.freqs[1]) - 500000.0 ** (-2 / 64)) < 1e-15
    layer.close()
    plain.close()


@pytest.mark.parametrize("hd,heads,dtype,window,fused", [(64, 4, "f32", None, False), (64, 4, "f16", (30, 0, 2), True), (80, 2, "bf16", None, False)])
def test_model_drafts_over_a_cache(ctx, hd, heads, dtype, window, fused):
    """A prompt, drafts of two sequences and accepted branches through Transformer.extend: every layer's attention against float64 over what the cache holds, which is its keys,
    turned, and values."""
    model, p = rotated_model(ctx, hd, heads, 2, 32, 4, (10000.0, None, "halves"), window, fused)
    cache, gen = K.PagedCache(ctx, pimdl, 2, 60, heads, hd, 16, dtype, 3, 200), gen_of(5)
    r = model.layers[0].rotary
    left, sinks = (1 << 40, 0) if window is None else (window[0], window[2])
    length = [0, 0, 0]
    for seqs, counts, drafted in (([0, 2], [50, 4], False), ([2, 0], [12, 33], True), ([0, 2], [1, 1], False), ([1, 0, 2], [17, 9, 30], True)):
        n, starts, lst = sum(counts), starts_of(counts), ints(*seqs)
        parents = forest(counts, 7) if drafted else ints(*[i - 1 for c in counts for i in range(c)])
        tree = None
        if drafted:
            tree = K.DraftTree(ctx, pimdl, n)
            tree.build(parents, starts)
        branches = split(parents, counts)
        x = randn(gen, n, p.token_dim)
        y = model.extend(x, cache, starts, lst, ints(*counts), tree=tree)
        torch.cuda.synchronize()
        assert int(cache.lacking) == 0
        h = x
        place = torch.tensor(np.concatenate([length[s] + np.array(depths_of(b)) for s, b in zip(seqs, branches)]), device="cuda")
        for i, layer in enumerate(model.layers):  # the same layers once more, stage by stage
            keep = {}
            h = layer.forward(h, keep, cached=(cache, i, starts, lst, tree))
            torch.cuda.synchronize()
            want_k, off_k = turned(keep["k"], place, r.freqs, "halves", hd)
            at = 0
            for s, c, b in zip(seqs, counts, branches):
                slots = torch.arange(length[s] + c, device="cuda")
                pages = cache.tables[s].long()[slots // 16]
                kk, vv = cache.k[i, pages, :, slots % 16], cache.v[i, pages, :, slots % 16]
                check_turned(kk[length[s]:].flatten(1), want_k[at:at + c], off_k[at:at + c], dtype)
                assert torch.equal(vv[length[s]:].flatten(1), keep["v"][at:at + c].to(TYPES[dtype]))
                want, off, mass = reference_tree(keep["q"][at:at + c].reshape(c, heads, hd), kk, vv, b, left, sinks, 1 / math.sqrt(hd))
                check(keep["attn"][at:at + c].reshape(c, heads, hd), want, off, mass, "f32")
                at += c
        assert torch.equal(h, y)
        if drafted:
            last, kept = [c // 2 for c in counts], torch.zeros(len(seqs), device="cuda", dtype=torch.int32)
            cache.accept(tree, ints(*last), kept, starts, lst)
            torch.cuda.synchronize()
            for s, b, e, m in zip(seqs, branches, last, kept.tolist()):
                assert m == depths_of(b)[e] + 1
                length[s] += m
        else:
            for s, c in zip(seqs, counts):
                length[s] += c
        assert cache.lengths.tolist() == length
    model.close()
