"""Refusals of the shaped-score, tree, multi-axis rotary and commit entry
points, on the CPU, before any device work."""
import ctypes

import numpy as np
import pytest
import torch

from nanovllm_amd import _native
from nanovllm_amd.kernels.scored import scored_attention
from nanovllm_amd.kernels.tree import (commit_tree_path, tree_attention, tree_mask_from_parents)
from nanovllm_amd.layers.rotary import pair_axes, qk_norm_mrope_store


def _scored(heads=8, kvh=2, dim=128, page=32, dtype=torch.bfloat16, pool=torch.bfloat16, **kw):
    q = torch.zeros(3, heads, dim, dtype=dtype)
    cache = torch.zeros(4, page, kvh, dim, dtype=pool)
    args = dict(scale=0.1, block_tables=torch.zeros(3, 1, dtype=torch.int32), num_decode_rows=3,
                decode_context_lens=torch.ones(3, dtype=torch.int32))
    args.update(kw)
    return scored_attention(q, cache, cache.clone(), **args)


@pytest.mark.parametrize("bad", [
    dict(dim=64), dict(page=48), dict(heads=9), dict(dtype=torch.float16), dict(pool=torch.int8),
    dict(scale=0.0), dict(scale=float("nan")), dict(softcap=-1.0), dict(softcap=float("inf")),
    dict(window=-1), dict(alibi_slopes=torch.zeros(7)), dict(num_decode_rows=2),
    dict(decode_context_lens=torch.ones(2, dtype=torch.int32)), dict(decode_context_lens=None),
    dict(block_tables=torch.zeros(2, 1, dtype=torch.int32)),
    dict(block_tables=torch.zeros(3, dtype=torch.int32)), dict(block_tables=None),
    dict(num_decode_rows=0, cu_seqlens_q_list=[0, 3], cu_seqlens_k_list=[0, 2]),
    dict(num_decode_rows=0, cu_seqlens_q_list=[0, 2], cu_seqlens_k_list=[0, 2]),
    dict(num_decode_rows=0, cu_seqlens_q_list=[0, 3], cu_seqlens_k_list=[0]),
    dict(num_decode_rows=0, cu_seqlens_q_list=[0, 3], cu_seqlens_k_list=[0, 3],
         prefix_lens=torch.ones(2, dtype=torch.int32)),
    dict(num_decode_rows=0, cu_seqlens_q_list=[0, 3], cu_seqlens_k_list=[0, 3], block_tables=None,
         k=torch.zeros(2, 2, 128, dtype=torch.bfloat16),
         v=torch.zeros(2, 2, 128, dtype=torch.bfloat16)),
])
def test_scored_attention_refuses(bad):
    with pytest.raises(ValueError):
        _scored(**bad)


def test_scored_attention_needs_device_tensors():
    with pytest.raises(RuntimeError, match="device"):
        _scored()


def _tree(heads=8, mask=None, **kw):
    q = torch.zeros(6, heads, 128, dtype=torch.bfloat16)
    cache = torch.zeros(4, 32, 2, 128, dtype=torch.bfloat16)
    mask = torch.ones(6, 1, dtype=torch.int64) if mask is None else mask
    return tree_attention(q, cache, cache.clone(), torch.zeros(2, 1, dtype=torch.int32),
                          kw.pop("context_lens", torch.ones(2, dtype=torch.int32)), mask,
                          kw.pop("scale", 0.1), **kw)


@pytest.mark.parametrize("bad", [
    dict(heads=9), dict(mask=torch.ones(5, 1, dtype=torch.int64)),
    dict(mask=torch.ones(6, 1, dtype=torch.int32)), dict(mask=torch.ones(6, dtype=torch.int64)),
    dict(mask=torch.ones(6, 0, dtype=torch.int64)), dict(context_lens=torch.ones(3)),
    dict(cu_seqlens_q=torch.tensor([0, 2, 6])),
    dict(cu_seqlens_q=torch.tensor([0, 6]), max_seqlen_q=6),
    dict(cu_seqlens_q=torch.tensor([0, 2, 6]), max_seqlen_q=65), dict(scale=-1.0),
    dict(softcap=-2.0), dict(window=-5),
])
def test_tree_attention_refuses(bad):
    with pytest.raises(ValueError):
        _tree(**bad)


def test_tree_attention_needs_device_tensors():
    with pytest.raises(RuntimeError, match="device"):
        _tree()


def test_tree_mask_from_parents():
    mask = tree_mask_from_parents([[-1, 0, 0, 1], [], [-1, -1, 1]])
    assert mask.tolist() == [[1], [3], [5], [11], [1], [2], [6]]
    chain = tree_mask_from_parents([list(range(-1, 69))])
    assert chain.shape == (70, 2) and chain[63].tolist() == [-1, 0]
    assert chain[69].tolist() == [-1, 63]
    assert tree_mask_from_parents([]).shape == (0, 1)
    for bad in ([[0]], [[-1, 1]], [[-2]]):
        with pytest.raises(ValueError):
            tree_mask_from_parents(bad)


def test_pair_axes():
    assert pair_axes((24, 20, 20), False).tolist() == [0] * 24 + [1] * 20 + [2] * 20
    mixed = pair_axes((24, 20, 20), True)
    assert [int((mixed == a).sum()) for a in range(3)] == [24, 20, 20]
    assert mixed[:6].tolist() == [0, 1, 2, 0, 1, 2] and mixed[60:].tolist() == [0, 0, 0, 0]
    for bad, inter in (((64, 1), False), ((), False), ((10, 30, 24), True), ((1,) * 64, False),
                       ((65, -1), False)):
        with pytest.raises(ValueError):
            pair_axes(bad, inter)


def _mrope(n=4, axes=3, **kw):
    bf = dict(dtype=torch.bfloat16)
    args = dict(q=torch.zeros(n, 8, 128, **bf), k=torch.zeros(n, 2, 128, **bf), v=None,
                positions=torch.zeros(axes, n, dtype=torch.int64),
                cos_sin_cache=torch.zeros(10, 128), sections=(24, 20, 20))
    args.update(kw)
    return qk_norm_mrope_store(**args)


@pytest.mark.parametrize("bad", [
    dict(axes=2), dict(positions=torch.zeros(12, dtype=torch.int64)), dict(sections=(32, 32)),
    dict(sections=(30, 20, 20)), dict(q=torch.zeros(4, 8, 64, dtype=torch.bfloat16)),
    dict(q=torch.zeros(4, 8, 128)), dict(k=torch.zeros(3, 2, 128, dtype=torch.bfloat16)),
    dict(q_norm_weight=torch.ones(64)), dict(k_cache=torch.zeros(1, 32, 2, 128)),
    dict(q_out=torch.zeros(4, 8, 64, dtype=torch.bfloat16)),
])
def test_mrope_refuses(bad):
    with pytest.raises(ValueError):
        _mrope(**bad)


def test_mrope_needs_device_tensors():
    with pytest.raises(RuntimeError, match="device"):
        _mrope()


@pytest.mark.parametrize("bad", [
    lambda a: a.update(kv_cache=torch.zeros(2, 3, 4)),
    lambda a: a.update(paths=torch.zeros(3, 2, dtype=torch.int32)),
    lambda a: a.update(context_lens=torch.zeros(3, dtype=torch.int32)),
    lambda a: a.update(path_lens=torch.zeros(1, dtype=torch.int32)),
    lambda a: a.update(block_tables=torch.zeros(2, dtype=torch.int32)),
])
def test_commit_refuses(bad):
    i32 = dict(dtype=torch.int32)
    args = dict(kv_cache=torch.zeros(2, 1, 4, 32, 2, 128), block_tables=torch.zeros(2, 1, **i32),
                context_lens=torch.zeros(2, **i32), paths=torch.zeros(2, 4, **i32),
                path_lens=torch.zeros(2, **i32))
    with pytest.raises(RuntimeError, match="device"):
        commit_tree_path(**args)
    bad(args)
    with pytest.raises(ValueError):
        commit_tree_path(**args)
    with pytest.raises(AssertionError):
        commit_tree_path(torch.zeros(2, 1, 4, 32, 2, 256)[..., ::2], torch.zeros(2, 1, **i32),
                         torch.zeros(2, **i32), torch.zeros(2, 4, **i32), torch.zeros(2, **i32))


def _c(name, *args):
    lib = _native.load()
    rc = getattr(lib, name)(*args)
    return rc, lib.kvc_last_error().decode()


def test_entry_points_refuse_before_any_launch():
    """Null pointers, bad sizes, misaligned rows and a small workspace come
    back as status codes (no device here: a launch would fail otherwise)."""
    buf = ctypes.create_string_buffer(4096)
    at = (ctypes.addressof(buf) + 255) // 256 * 256

    def scored(q=at, kvh=2, hd=128, k=at, page=32, tables=at, dec=1, lens=at, prefill=0, cap=0.0,
               window=0, scale=0.1, out=at, ws=at, ws_bytes=0, heads=8, blocks=4, width=1):
        return _c("kvc_scored_attention", q, heads * 128, 128, 1, heads, k, k, blocks, page, kvh,
                  hd, None, 0, 0, None, 0, 0, 0, tables, 1, width, dec, lens, prefill, None, None,
                  1, None, None, cap, window, scale, out, heads * 128, 128, ws, ws_bytes, None)

    for kw, rc in ((dict(hd=64), -1), (dict(kvh=3), -1), (dict(kvh=0), -1), (dict(scale=0.0), -1),
                   (dict(cap=-1.0), -1), (dict(window=-1), -1), (dict(q=None), -1),
                   (dict(out=None), -1), (dict(q=at + 8), -2), (dict(k=None), -1),
                   (dict(k=at + 2), -2), (dict(page=16), -1), (dict(page=0), -1),
                   (dict(blocks=0), -1), (dict(width=1 << 40), -1), (dict(lens=None), -1),
                   (dict(dec=2), -1), (dict(dec=-1), -1), (dict(tables=None), -1),
                   (dict(dec=0, prefill=1), -1), (dict(heads=1024), -1), (dict(), -4),
                   (dict(ws=None, ws_bytes=1 << 40), -4)):
        got, msg = scored(**kw)
        assert got == rc and msg, (kw, got, msg)

    def tree(mask=at, words=1, cu=None, most=1, tokens=1, batch=1, lens=at):
        return _c("kvc_tree_attention", at, 1024, 128, tokens, 8, at, at, 4, 32, 2, 128, at, 1, 1,
                  batch, lens, cu, most, mask, words, None, 0.0, 0, 0.1, at, 1024, 128, at, 0,
                  None)

    for kw, rc in ((dict(mask=None), -1), (dict(words=0), -1), (dict(most=65, tokens=65), -1),
                   (dict(tokens=2), -1), (dict(lens=None), -1), (dict(), -4),
                   (dict(batch=-1), -1), (dict(batch=0, tokens=0), 0)):
        got, msg = tree(**kw)
        assert got == rc, (kw, got, msg)

    axes = np.zeros(64, dtype=np.int32)

    def mrope(n=1, naxes=3, ax=axes.ctypes.data, q=at, pos=at, pb=8, kc=None, vc=None, hd=128):
        return _c("kvc_qk_norm_mrope_store", q, 1024, 128, at, 256, 128, at, 256, 128, n, 8, 2, hd,
                  pos, n, pb, naxes, ax, None, None, 1e-6, at, 10, at, 1024, 128, None, 0, 0, kc,
                  vc, 4, None, 4, None)

    for kw, rc in ((dict(hd=64), -1), (dict(n=-1), -1), (dict(naxes=0), -1), (dict(naxes=5), -1),
                   (dict(ax=None), -1), (dict(pb=2), -1), (dict(q=None), -1), (dict(pos=None), -1),
                   (dict(q=at + 2), -2), (dict(kc=at), -1), (dict(kc=at, vc=at), -1),
                   (dict(n=0), 0)):
        got, msg = mrope(**kw)
        assert got == rc, (kw, got, msg)
    far = axes.copy()
    far[5] = 3
    assert mrope(ax=far.ctypes.data)[0] == -1
    far[5] = -1
    assert mrope(ax=far.ctypes.data)[0] == -1

    def commit(pool=at, planes=1, stride=4 * 32 * 64, blocks=4, page=32, row=64, batch=1, most=4,
               paths=at):
        return _c("kvc_commit_rows", pool, planes, stride, blocks, page, row, at, 1, 1, at, paths,
                  4, most, at, batch, None)

    for kw, rc in ((dict(pool=None), -1), (dict(planes=-1), -1), (dict(blocks=0), -1),
                   (dict(page=0), -1), (dict(row=0), -1), (dict(stride=64), -1),
                   (dict(paths=None), -1), (dict(batch=0), 0), (dict(most=0), 0),
                   (dict(planes=0), 0)):
        got, msg = commit(**kw)
        assert got == rc, (kw, got, msg)


def test_caps_and_scales_that_fp32_cannot_divide():
    """scale / softcap past fp32 would make 0 x inf of a zero logit."""
    buf = ctypes.create_string_buffer(4096)
    at = (ctypes.addressof(buf) + 255) // 256 * 256
    for cap, scale, rc in ((1e-38, 100.0, -1), (0.0, 3e38, -1), (1e-30, 0.1, -4), (1e30, 0.1, -4)):
        got, msg = _c("kvc_scored_attention", at, 1024, 128, 1, 8, at, at, 4, 32, 2, 128, None, 0,
                      0, None, 0, 0, 0, at, 1, 1, 1, at, 0, None, None, 1, None, None, cap, 0,
                      scale, at, 1024, 128, at, 0, None)
        assert got == rc and msg, (cap, scale, got, msg)


def test_a_layers_slopes_move_with_it():
    from nanovllm_amd.layers.attention import Attention
    layer = Attention(8, 128, 0.1, 2, alibi_slopes=torch.ones(8))
    assert dict(layer.named_buffers())["alibi_slopes"] is layer.alibi_slopes
    assert not layer.state_dict()
    assert layer.to("meta").alibi_slopes.device.type == "meta"
    assert Attention(8, 128, 0.1, 2).alibi_slopes is None


@pytest.mark.parametrize("out", [torch.zeros(2, 8, 128, dtype=torch.bfloat16),
                                 torch.zeros(3, 8, 128),
                                 torch.zeros(3, 8, 132, dtype=torch.bfloat16)[..., 4:]])
def test_scored_attention_refuses_other_outputs(out):
    with pytest.raises(ValueError, match="out must be"):
        _scored(out=out)


def test_graph_runner_checks_score_shapes():
    from nanovllm_amd.engine.graph_runner import DecodeGraphRunner
    caches = [torch.zeros(3, 32, 2, 128, dtype=torch.bfloat16) for _ in range(2)]
    for bad in ([dict(window=3)], dict(cap=50.0), [dict(), dict(prefix_lens=None)]):
        with pytest.raises(ValueError, match="score shape"):
            DecodeGraphRunner(caches, caches, 8, 2, 2, 0.1, score_shapes=bad)
    one = dict(window=3)
    runner = DecodeGraphRunner(caches, caches, 8, 2, 2, 0.1, score_shapes=[None, one])
    assert runner.score_shapes == [{}, one]
    assert DecodeGraphRunner(caches, caches, 8, 2, 2, 0.1, score_shapes=one).score_shapes == [one] * 2


@pytest.mark.parametrize("bad", [
    dict(cu_seqlens_q_list=[5, 8], cu_seqlens_k_list=[0, 3]),     # a slice of a larger batch
    dict(cu_seqlens_q_list=[2, 5], cu_seqlens_k_list=[2, 5]),
    dict(cu_seqlens_q_list=[-1, 2], cu_seqlens_k_list=[0, 3]),
    dict(cu_seqlens_q=torch.tensor([5, 8]), cu_seqlens_k=torch.tensor([0, 3])),
    dict(cu_seqlens_q_list=[0, 3], cu_seqlens_k_list=[-3, 0]),
    dict(cu_seqlens_q_list=[0, 3], cu_seqlens_k_list=[-1, 2], block_tables=None,
         k=torch.zeros(2, 2, 128, dtype=torch.bfloat16),
         v=torch.zeros(2, 2, 128, dtype=torch.bfloat16)),
    dict(cu_seqlens_q_list=[], cu_seqlens_k_list=[]),
])
def test_offsets_that_do_not_start_at_the_first_row(bad):
    """cu_seqlens_q are rows of this q: the kernel would leave those before the
    first offset unwritten and cut the last sequence."""
    with pytest.raises(ValueError):
        _scored(num_decode_rows=0, **bad)


def test_a_layers_slopes_stay_fp32():
    """Casting the model does not round them, whichever way it is cast; moved
    and cast at once, they move."""
    from nanovllm_amd.layers.attention import Attention
    slopes = torch.tensor([2.0 ** (-8.0 * (i + 1) / 12) for i in range(12)])
    for cast in (lambda m: m.to(torch.bfloat16), lambda m: m.half(), lambda m: m.double(),
                 lambda m: m.bfloat16().float(), lambda m: m.to("cpu", torch.bfloat16)):
        model = torch.nn.Sequential(torch.nn.Linear(2, 2),
                                    Attention(12, 128, 0.1, 2, alibi_slopes=slopes.clone()))
        assert cast(model) is model
        layer = model[1]
        assert layer.alibi_slopes.dtype == torch.float32
        assert torch.equal(layer.alibi_slopes, slopes)
        assert dict(layer.named_buffers())["alibi_slopes"] is layer.alibi_slopes
    moved = Attention(12, 128, 0.1, 2, alibi_slopes=slopes).to("meta", torch.bfloat16)
    assert moved.alibi_slopes.device.type == "meta"
    assert moved.alibi_slopes.dtype == torch.float32
    given = Attention(12, 128, 0.1, 2, alibi_slopes=slopes.double()).alibi_slopes
    assert given.dtype == torch.float32 and torch.equal(given, slopes)
    assert Attention(12, 128, 0.1, 2).to(torch.bfloat16).alibi_slopes is None


def _bound(monkeypatch, *layers):
    from nanovllm_amd.engine import kv_runner
    monkeypatch.setattr(kv_runner, "BlockMover", lambda pool: None)     # (needs a GPU pool)
    kv = kv_runner.KVCacheRunner(len(layers), 2, 32, 2, 128, device="cpu")
    assert kv.bind(layers) == len(layers)
    return kv


def test_graph_runner_takes_the_bound_layers_shapes(monkeypatch):
    """A shaped layer is captured shaped without being named again."""
    from nanovllm_amd.engine.graph_runner import DecodeGraphRunner
    from nanovllm_amd.layers.attention import Attention
    slopes = torch.ones(8)
    layers = [Attention(8, 128, 0.1, 2), Attention(8, 128, 0.1, 2, softcap=50.0, window=7),
              Attention(8, 128, 0.1, 2, alibi_slopes=slopes)]
    kv = _bound(monkeypatch, *layers)
    got = DecodeGraphRunner.from_kv_runner(kv, 8, 2, 2, 0.1).score_shapes
    assert got[0] == {}
    assert got[1] == dict(softcap=50.0, alibi_slopes=None, window=7)
    assert got[2]["alibi_slopes"] is layers[2].alibi_slopes and not got[2]["softcap"]
    plain = DecodeGraphRunner.from_kv_runner(kv, 8, 2, 2, 0.1, score_shapes={})
    assert plain.score_shapes == [{}] * 3
    one = dict(window=3)
    assert DecodeGraphRunner.from_kv_runner(kv, 8, 2, 2, 0.1,
                                            score_shapes=one).score_shapes == [one] * 3
    assert _bound(monkeypatch, Attention(8, 128, 0.1, 2)).score_shapes() == [None]


@pytest.mark.parametrize("bad", [dict(softcap=-1.0), dict(window=-2),
                                 dict(alibi_slopes=torch.ones(7)),
                                 dict(alibi_slopes=torch.ones(8, device="meta"))])
def test_graph_runner_checks_values_before_a_capture(bad):
    from nanovllm_amd.engine.graph_runner import DecodeGraphRunner
    caches = [torch.zeros(3, 32, 2, 128, dtype=torch.bfloat16)]
    with pytest.raises(ValueError):
        DecodeGraphRunner(caches, caches, 8, 2, 2, 0.1, score_shapes=bad)


def test_pair_axes_belong_to_the_caller():
    """Writing to them changes no later call's."""
    from nanovllm_amd.layers.rotary import _pair_axes_at
    held, at = _pair_axes_at((16, 24, 24), False)
    axes = pair_axes((16, 24, 24), False)
    assert axes.ctypes.data != at and axes.tolist() == held.tolist()
    axes[0] = 2
    assert pair_axes((16, 24, 24), False)[0] == 0 and held[0] == 0
    assert _pair_axes_at((16, 24, 24), False)[1] == at
