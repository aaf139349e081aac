"""Host logic of serving that needs no GPU: what Transformer.extend and PagedCache refuse, and that a refused call has changed nothing.  Stand-ins
record what would have been launched."""
import os

import pytest
import torch
import yaml

from __graft_entry__ import load_package

pimdl = load_package()
from pim_dl_asplos_amd import kvcache as K  # noqa: E402
from pim_dl_asplos_amd import transformer as T  # noqa: E402


class Recorder:
    """Takes any call of the library's binding and says that it went well."""

    def __init__(self):
        self.calls = []

    def __getattr__(self, name):
        return lambda *a: self.calls.append(name) or 0


def params(window=None, heads=4, hd=64):
    p = T.TransformerParams(8, 2, heads, hd, heads * hd, 2 * heads * hd, 2)
    p.window = window
    return p


def context(stream=None):
    c = pimdl.Context.__new__(pimdl.Context)
    c._h, c.stream = None, stream
    return c


def cache_of(ctx, layers=2, heads=4, hd=64, page_tokens=16, seqs=3):
    c = K.PagedCache.__new__(K.PagedCache)
    c.ctx, c._lib, c._unlimited, c._book = ctx, Recorder(), pimdl.UNLIMITED, None
    c.layers, c.kv_heads, c.head_dim, c.page_tokens = layers, heads, hd, page_tokens
    c.k = torch.zeros(layers, 2, heads, page_tokens, hd)
    c.tables = torch.full((seqs, 4), -1, dtype=torch.int32)
    c._layer = [None] * layers
    return c


def model_of(ctx, p, layers=2):
    made = []
    for _ in range(layers):
        layer = T.TransformerLayer.__new__(T.TransformerLayer)
        layer.ctx, layer.params, layer.torch, layer._max_tokens, layer._unlimited = ctx, p, torch, p.n, pimdl.UNLIMITED
        made.append(layer)
    return T.Transformer.from_layers(made, p)


def ints(*x):
    return torch.tensor(x, dtype=torch.int32)


class Reached(Exception):
    pass


def extend(monkeypatch, model, cache, x=None, starts=None, seqs=None, counts=None):
    """extend() up to the first layer's kernels."""
    def run(self, *a):
        raise Reached

    monkeypatch.setattr(T.TransformerLayer, "_run", run)
    for layer in model.layers:
        layer.side, layer.fused_qkv, layer.qkv_group = None, True, None
    return model.extend(torch.zeros(3, 256) if x is None else x, cache, ints(0, 2, 3) if starts is None else starts, ints(0, 2) if seqs is None else seqs,
                        ints(2, 1) if counts is None else counts)


def test_extend_reserves_and_runs(monkeypatch):
    ctx = context()
    for window in (None, (5, 0, 1), (None, 0, 0)):
        cache = cache_of(ctx, layers=3)  # (a layer more than the model)
        with pytest.raises(Reached):
            extend(monkeypatch, model_of(ctx, params(window)), cache)
        assert cache._lib.calls == ["pimdl_pages_reserve"]


def test_extend_without_tokens_reserves_and_returns(monkeypatch):
    ctx = context()
    cache, x = cache_of(ctx), torch.zeros(0, 256)
    assert extend(monkeypatch, model_of(ctx, params()), cache, x=x, starts=ints(0, 0, 0), counts=ints(0, 0)) is x
    assert cache._lib.calls == ["pimdl_pages_reserve"]


@pytest.mark.parametrize("window,cache,call,text", [
    ((4, 4, 0), {}, {}, "right = 0"),
    ((4, None, 0), {}, {}, "right = 0"),
    (None, dict(layers=1), {}, "no layer 1"),
    (None, dict(heads=2), {}, "2 heads of 64"),
    (None, dict(hd=32), {}, "4 heads of 32"),
    (None, dict(page_tokens=24), {}, "power of two"),
    (None, {}, dict(x=torch.zeros(3, 255)), r"\[tokens\]\[256\]"),
    (None, {}, dict(x=torch.zeros(3, 256, dtype=torch.float16)), "float32"),
    (None, {}, dict(x=torch.zeros(768)), "float32"),
    (None, {}, dict(x=torch.zeros(17, 256)), "built for 16"),
    (None, {}, dict(x=torch.zeros(3, 256, device="meta")), "the cache's GPU"),
    (None, {}, dict(starts=ints(0, 3)), "one number more"),
    (None, {}, dict(starts=torch.tensor([0, 2, 3])), "int32"),
    (None, {}, dict(starts=ints(0, 2, 3).to("meta")), "the cache's GPU"),
    (None, {}, dict(seqs=ints(0, 1, 2)), "one number more"),
    (None, {}, dict(counts=ints(3)), "one length"),
    (None, {}, dict(counts=torch.tensor([2, 1])), "int32"),
])
def test_a_refused_extend_leaves_the_book_alone(monkeypatch, window, cache, call, text):
    ctx = context()
    c = cache_of(ctx, **cache)
    with pytest.raises(ValueError, match=text):
        extend(monkeypatch, model_of(ctx, params(window)), c, **call)
    assert c._lib.calls == []


def test_heads_beyond_the_kernels_are_refused_first(monkeypatch):
    ctx = context()
    c = cache_of(ctx, heads=1, hd=260)
    with pytest.raises(ValueError, match="up to 256"):
        extend(monkeypatch, model_of(ctx, params(heads=1, hd=260)), c, x=torch.zeros(3, 260))
    assert c._lib.calls == []


def test_a_cache_on_another_stream_is_refused(monkeypatch):
    """Two contexts: their calls are in order only where both were given the same stream."""
    for own, other, fine in ((None, None, False), (7, None, False), (None, 7, False), (7, 8, False), (7, 7, True)):
        cache = cache_of(context(other))
        with pytest.raises(Reached if fine else ValueError, match=None if fine else "another stream"):
            extend(monkeypatch, model_of(context(own), params()), cache)
        assert cache._lib.calls == (["pimdl_pages_reserve"] if fine else [])


WINDOW = dict(q=1, k=1, v=1, out=1, starts=1, batch=1, tokens=4, heads=2, kv_heads=1, head_dim=64, q_stride=128, kv_stride=64, out_stride=128, left=5, right=0,
              sinks=1, scale=1.0)


@pytest.mark.parametrize("name", ["left", "right", "sinks", "batch", "tokens", "heads", "kv_heads", "head_dim", "q_stride", "kv_stride", "out_stride", "dtype"])
def test_numbers_that_32_bits_do_not_hold_are_refused(monkeypatch, name):
    """-1 would become no border, 2^32 none at all."""
    monkeypatch.setattr(pimdl, "lib", lambda: pytest.fail("the library was called"))
    for bad in (-1, -2 ** 31, 2 ** 32, 2 ** 32 + 5):
        with pytest.raises(ValueError, match=name):
            context().attention_window_ptr(**(WINDOW | {name: bad}))


def test_attend_refuses_numbers_that_32_bits_do_not_hold():
    c, q = cache_of(context()), torch.zeros(2, 256)
    for bad in (dict(left=-1), dict(left=2 ** 32), dict(sinks=-1), dict(sinks=2 ** 32 + 1)):
        with pytest.raises(ValueError, match=list(bad)[0]):
            c.attend(0, q, torch.zeros(2, 256), ints(0, 1, 2), 4, **bad)
    far = torch.empty_strided((2, 256), (2 ** 32 + 256, 1), device="meta")
    with pytest.raises(ValueError, match="stride"):
        c.attend(0, far, far, ints(0, 1, 2), 4)
    assert c._lib.calls == []
    c.attend(0, q, torch.zeros(2, 256), ints(0, 1, 2), 4, left=0xFFFFFFFF, sinks=3)
    c.attend(0, q[:1], torch.zeros(1, 256), ints(0, 1), 4, left=0)
    assert c._lib.calls == ["pimdl_attention_paged"] * 2


@pytest.mark.parametrize("window", [(-1, 0, 0), (3, -2, 0), (3, 0, -1), (2 ** 32, 0, 0), (None, 2 ** 32, 0), (None, None, 2 ** 40)])
def test_windows_out_of_range_are_refused(monkeypatch, window):
    ctx = context()
    cache = cache_of(ctx)
    with pytest.raises(ValueError, match="window"):
        params(window).borders()
    with pytest.raises(ValueError, match="window"):
        extend(monkeypatch, model_of(ctx, params(window)), cache)
    assert cache._lib.calls == []
    with pytest.raises(TypeError):
        params((1.5, 0, 0)).borders()
    assert params((None, 7, 2)).borders() == (pimdl.UNLIMITED, 7, 2)


def test_a_configuration_with_a_window_out_of_range_is_refused(tmp_path):
    cfg = yaml.safe_load(open(os.path.join(os.path.dirname(__file__), "golden", "transformer_small.yaml")))
    for window, fine in (([5, None, 1], True), ([-5, 0, 1], False), ([5, 0, 1 << 32], False)):
        cfg["network_params"]["attention_window"] = window
        path = tmp_path / "w.yaml"
        path.write_text(yaml.safe_dump(cfg))
        if fine:
            assert T.TransformerParams.from_yaml(path).window == (5, None, 1)
        else:
            with pytest.raises(ValueError, match="window"):
                T.TransformerParams.from_yaml(path)


@pytest.mark.parametrize("layer", [-1, -2, 2, 7])
def test_layers_that_are_not_there_are_refused(layer):
    c, x = cache_of(context()), torch.zeros(2, 256)
    with pytest.raises(IndexError, match="layer"):
        c.append(layer, x, x, ints(0, 1, 2))
    with pytest.raises(IndexError, match="layer"):
        c.attend(layer, x, torch.zeros(2, 256), ints(0, 1, 2), 4)
    assert c._lib.calls == []
    c.append(1, x, x, ints(0, 1, 2))
    assert c._lib.calls == ["pimdl_cache_append"]
