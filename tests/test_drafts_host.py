"""Host logic of rotated positions and drafted trees that needs no GPU: what Rotary, DraftTree, PagedCache and Transformer.extend refuse, and that a refused call has launched
nothing.  Stand-ins record what would have been launched."""
import os

import pytest
import torch
import yaml

from __graft_entry__ import load_package
from test_serving_host import Reached, Recorder, cache_of, context, extend, ints, model_of, params

pimdl = load_package()
from pim_dl_asplos_amd import kvcache as K  # noqa: E402
from pim_dl_asplos_amd import transformer as T  # noqa: E402


@pytest.fixture(autouse=True)
def recorder(monkeypatch):
    r = Recorder()
    monkeypatch.setattr(pimdl, "lib", lambda: r)
    return r


def freqs(n):
    return torch.ones(n, dtype=torch.float64)


def rotary_of(hd=64, n=32, pairs="halves"):
    return K.Rotary(context(), pimdl, hd, freqs=freqs(n), pairs=pairs)


def tree_of(tokens=8, words=1, ctx=None):
    return K.DraftTree.over(ctx or context(), pimdl, torch.zeros(tokens, words, dtype=torch.int32), torch.zeros(tokens, dtype=torch.int32))


@pytest.mark.parametrize("kw,text", [
    (dict(pairs="thirds"), "halves"), (dict(dims=63), "even"), (dict(dims=66), "even"), (dict(dims=0), "even"), (dict(base=0.0), "base"), (dict(base=float("inf")), "base"),
    (dict(base=float("nan")), "base"), (dict(freqs=freqs(33)), "float64"), (dict(freqs=freqs(0)), "float64"), (dict(freqs=torch.ones(32)), "float64"),
    (dict(freqs=freqs(64)[::2]), "float64"), (dict(freqs=freqs(32).reshape(4, 8)), "float64"), (dict(freqs=freqs(16), dims=64), "16 frequencies"),
])
def test_rotations_that_cannot_be_are_refused(kw, text):
    with pytest.raises(ValueError, match=text):
        K.Rotary(context(), pimdl, 64, **kw)


def test_rotate_refuses_what_does_not_fit(recorder):
    r, q, k, at = rotary_of(), torch.zeros(3, 256), torch.zeros(3, 128), ints(0, 3)
    for bad, text in (((q, k, q[:2], k, at), "one shape"), ((q, k, q, k[:, :64], at), "one shape"), ((q, k[:2], q, k[:2], at), "number of rows"),
                      ((q, k, q.half(), k, at), "one type"), ((q, k.half(), q, k.half(), at), "one type"), ((q[:, :250], k, q[:, :250], k, at), "heads"),
                      ((q, k, q, k, at.long()), "int32"), ((q, k, q, k, at[:0]), "one number more"), ((q.int(), k.int(), q.int(), k.int(), at), "unit column"),
                      ((torch.zeros(256, 3).t(), k, q, k, at), "unit column"), ((q[0], k, q[0], k, at), "number of rows|one shape|heads")):
        with pytest.raises((ValueError, IndexError), match=text):
            r.rotate(*bad)
    assert recorder.calls == []
    r.rotate(q, k, q, k, at)
    r.rotate(q, k[:, :0], q, k[:, :0], at)  # (queries alone)
    assert recorder.calls == ["pimdl_rotate"] * 2


def test_trees_that_cannot_be_are_refused(recorder):
    m, d = torch.zeros(4, 2, dtype=torch.int32), torch.zeros(4, dtype=torch.int32)
    for bad, text in (((m.long(), d), "int32"), ((m, d[:3]), "int32"), ((m, d.long()), "int32"), ((m[:, 0], d), "int32"), ((torch.zeros(4, 33, dtype=torch.int32), d), "1 to 32"),
                      ((m[:, :0], d), "1 to 32"), ((torch.zeros(4, 4, dtype=torch.int32)[:, ::2], d), "contiguous"), ((m, d.to("meta")), "one GPU")):
        with pytest.raises(ValueError, match=text):
            K.DraftTree.over(context(), pimdl, *bad)
    for tokens, most in ((-1, 4), (4, 0), (4, 1025)):
        with pytest.raises(ValueError, match="1 to 1024"):
            K.DraftTree(context(), pimdl, tokens, most)
    t = tree_of(4)
    for parents, starts, text in ((ints(-1, 0, 1, 2, 3), ints(0, 5), "room for 4"), (ints(-1).long(), ints(0, 1), "parents"), (ints(-1), ints(0, 1).long(), "starts"),
                                  (ints(-1), ints(), "one number more")):
        with pytest.raises(ValueError, match=text):
            t.build(parents, starts)
    assert recorder.calls == []
    t.build(ints(-1, 0), ints(0, 2))
    assert recorder.calls == ["pimdl_tree_build"]


def test_append_refuses_queries_and_rotations_that_do_not_fit():
    c, x, q, at = cache_of(context()), torch.zeros(2, 256), torch.zeros(2, 512), ints(0, 1, 2)
    for kw, text in ((dict(rotary=rotary_of(32, 16)), "heads of 32"), (dict(rotary=rotary_of(), q=q), "q_out"), (dict(rotary=rotary_of(), q=q, q_out=q[:1]), "one shape"),
                     (dict(rotary=rotary_of(), q=q.half(), q_out=q.half()), "type"), (dict(rotary=rotary_of(), q=q[:1], q_out=q[:1]), "number of rows"),
                     (dict(rotary=rotary_of(), q=q[:, :500], q_out=q[:, :500]), "heads"), (dict(rotary=rotary_of(), tree=tree_of(1)), "room for 1"), (dict(q=q, q_out=q), "none is given")):
        with pytest.raises(ValueError, match=text):
            c.append(0, x, x, at, **kw)
    with pytest.raises(IndexError):
        c.append(2, x, x, at, rotary=rotary_of())
    assert c._lib.calls == []
    c.append(0, x, x, at, rotary=rotary_of())
    c.append(1, x, x, at, rotary=rotary_of(), q=q, q_out=q, tree=tree_of(2))
    assert c._lib.calls == ["pimdl_cache_append_rotary"] * 2


def test_attend_and_accept_refuse_trees_and_lists_that_do_not_fit():
    c, q, at = cache_of(context()), torch.zeros(2, 256), ints(0, 1, 2)
    with pytest.raises(ValueError, match="room for 1"):
        c.attend(0, q, torch.zeros(2, 256), at, 4, tree=tree_of(1))
    c._row_bytes = 128
    for last, kept, starts, text in ((ints(0), ints(0, 0), at, "a number for each"), (ints(0, 0), ints(0), at, "a number for each"), (ints(0, 0).long(), ints(0, 0), at, "last"),
                                     (ints(0, 0), ints(0, 0).long(), at, "kept"), (ints(0, 0), ints(0, 0), at.long(), "starts")):
        with pytest.raises(ValueError, match=text):
            c.accept(tree_of(), last, kept, starts)
    assert c._lib.calls == []
    c.attend(0, q, torch.zeros(2, 256), at, 4, tree=tree_of(2))
    c.accept(tree_of(), ints(0, -1), ints(0, 0), at)
    assert c._lib.calls == ["pimdl_attention_tree", "pimdl_pages_accept"]


def run_extend(monkeypatch, model, cache, tree):
    def run(self, *a):
        raise Reached

    monkeypatch.setattr(T.TransformerLayer, "_run", run)
    for layer in model.layers:
        layer.side, layer.fused_qkv, layer.qkv_group = None, True, None
    return model.extend(torch.zeros(3, 256), cache, ints(0, 2, 3), ints(0, 2), ints(2, 1), tree=tree)


def test_extend_refuses_a_tree_before_it_makes_room(monkeypatch):
    ctx = context(5)
    for tree, text in ((tree_of(2, ctx=ctx), "room for 2"), (tree_of(ctx=context()), "another stream"), (tree_of(ctx=context(6)), "another stream")):
        cache = cache_of(ctx)
        with pytest.raises(ValueError, match=text):
            run_extend(monkeypatch, model_of(ctx, params()), cache, tree)
        assert cache._lib.calls == []
    cache, away = cache_of(ctx), tree_of(ctx=ctx)
    away.masks = away.masks.to("meta")
    with pytest.raises(ValueError, match="the cache's GPU"):
        run_extend(monkeypatch, model_of(ctx, params()), cache, away)
    assert cache._lib.calls == []
    with pytest.raises(Reached):
        run_extend(monkeypatch, model_of(ctx, params()), cache, tree_of(ctx=context(5)))
    assert cache._lib.calls == ["pimdl_pages_reserve"]


@pytest.mark.parametrize("rotary,fine", [([10000.0, 6, "halves"], True), ([500000, None, "neighbours"], True), ([0, 8, "halves"], False), ([1e4, 7, "halves"], False),
                                         ([1e4, 10, "halves"], False), ([1e4, 8, "thirds"], False), ([1e4, 8], False), (["nan", 8, "halves"], False)])
def test_a_configuration_with_a_rotation(tmp_path, rotary, fine):
    cfg = yaml.safe_load(open(os.path.join(os.path.dirname(__file__), "golden", "transformer_small.yaml")))
    cfg["network_params"]["rotary"] = rotary
    path = tmp_path / "r.yaml"
    path.write_text(yaml.safe_dump(cfg))
    if fine:
        p = T.TransformerParams.from_yaml(path)
        assert p.turns() == {"base": float(rotary[0]), "dims": rotary[1] or p.head_dim, "pairs": rotary[2]}
    else:
        with pytest.raises(ValueError):
            T.TransformerParams.from_yaml(path)


def test_a_model_without_a_rotation_reads_as_before():
    p = T.TransformerParams.from_yaml(os.path.join(os.path.dirname(__file__), "golden", "transformer_small.yaml"))
    assert p.rotary is None and T.TransformerLayer.rotary is None


def named_context(calls, name, stream=None):
    c = context(stream)
    c._h = name  # (of a context that is not closed)
    c.synchronize = lambda: calls.append(name)
    return c


def uses_of(c, tree):
    q, at = torch.zeros(2, 256), ints(0, 1, 2)
    c._row_bytes = 128
    return (lambda: c.append(0, q, q, at, rotary=rotary_of(), tree=tree), lambda: c.attend(0, q, torch.zeros(2, 256), at, 4, tree=tree),
            lambda: c.accept(tree, ints(0, -1), ints(0, 0), at))


@pytest.mark.parametrize("mine,its", [(5, 6), (5, None), (None, 6)])
def test_a_tree_on_another_stream_than_the_caches_is_refused(mine, its):
    c = cache_of(context(mine))
    for call in uses_of(c, tree_of(ctx=context(its))):
        with pytest.raises(ValueError, match="another stream"):
            call()
    assert c._lib.calls == []
    for call in uses_of(c, tree_of(ctx=context(mine) if mine else c.ctx)):
        call()
    assert c._lib.calls == ["pimdl_cache_append_rotary", "pimdl_attention_tree", "pimdl_pages_accept"]


def test_a_tree_between_two_contexts_with_streams_of_their_own(recorder):
    """Nobody else can order them: what reads the tree waits for what has filled it, and what fills it again for all that have read it."""
    log = []
    ours, other, its = (named_context(log, n) for n in ("ours", "other", "its"))
    tree, a, b = tree_of(ctx=its), cache_of(ours), cache_of(other)
    recorder.calls = a._lib.calls = b._lib.calls = log
    for c in (a, b):
        for call in uses_of(c, tree):
            call()
    reads = ["its", "pimdl_cache_append_rotary", "its", "pimdl_attention_tree", "its", "pimdl_pages_accept"]
    assert log == reads * 2
    log.clear()
    tree.build(ints(-1, 0), ints(0, 2))
    assert sorted(log[:2]) == ["other", "ours"] and log[2:] == ["pimdl_tree_build"]
    log.clear()
    tree.build(ints(-1, 0), ints(0, 2))  # (nobody has read it since)
    uses_of(cache_of(its), tree)[1]()    # its own context's
    assert log == ["pimdl_tree_build"]


def test_append_drops_no_argument_in_silence():
    c, x, q, at = cache_of(context()), torch.zeros(2, 256), torch.zeros(2, 512), ints(0, 1, 2)
    tree = tree_of(2, ctx=c.ctx)
    for kw, text in ((dict(rotary=rotary_of(), q_out=q), "no queries"), (dict(q_out=q), "none is given"), (dict(tree=tree_of(1, ctx=c.ctx)), "room for 1"),
                     (dict(tree=tree_of(2, ctx=context(5))), "another stream")):
        with pytest.raises(ValueError, match=text):
            c.append(0, x, x, at, **kw)
    assert c._lib.calls == []
    c.append(0, x, x, at, tree=tree)  # (a tree's keys have the places of any others)
    c.append(0, x, x, at, rotary=rotary_of(), q_out=q[:, :0])  # (no columns: nothing is dropped)
    assert c._lib.calls == ["pimdl_cache_append", "pimdl_cache_append_rotary"]


@pytest.mark.parametrize("base", [5e-324, 1e-310, 1e-300, 2.0 ** -30, -1.0])
def test_bases_whose_angles_are_lost_are_refused(base):
    """Frequencies beyond 2^21 radians a position take angles to where neighbouring doubles are a radian and more apart."""
    with pytest.raises(ValueError, match="base"):
        K.Rotary(context(), pimdl, 128, base=base)
    p = params(hd=128)
    p.rotary = (base, None, "halves")
    with pytest.raises(ValueError, match="base"):
        p.turns()
    p.rotary = (2.0 ** -21, None, "halves")
    assert p.turns()["base"] ** (-126 / 128) < 2.0 ** 21


@pytest.mark.parametrize("rotary", [10000.0, "halves", [1e4, 8.0, "halves"], [1e4, "8", "halves"], [[1e4], 8, "halves"], [1e4, 8, ["halves"]], {"base": 1e4}, []])
def test_a_configuration_without_a_rotation_or_with_none_that_can_be(tmp_path, rotary):
    cfg = yaml.safe_load(open(os.path.join(os.path.dirname(__file__), "golden", "transformer_small.yaml")))
    path = tmp_path / "r.yaml"
    cfg["network_params"]["rotary"] = None  # null: no rotation, as if it were not there
    path.write_text(yaml.safe_dump(cfg))
    assert T.TransformerParams.from_yaml(path).rotary is None
    cfg["network_params"]["rotary"] = rotary
    path.write_text(yaml.safe_dump(cfg))
    with pytest.raises(ValueError, match="rotary="):
        T.TransformerParams.from_yaml(path)
