"""Refusals of the 4-bit KV pool's entry points and of the step tables, on the CPU,
before any device work; and the 4-bit oracle against values worked out by hand."""
import ctypes

import numpy as np
import pytest
import torch

from nanovllm_amd import _native
from nanovllm_amd.engine.device_tables import DeviceBlockTables
from nanovllm_amd.engine.graph_runner import DecodeGraphRunner
from nanovllm_amd.engine.kv_runner import KVCacheRunner
from nanovllm_amd.kernels.kv_fp4 import (dequant_fp4, paged_decode_append_fp4, paged_decode_fp4,
                                         store_kvcache_fp4)
from nanovllm_amd.kernels.paged_attention import paged_decode_attention
from nanovllm_amd.kernels.step_tables import build_step_tables, new_step_tables
from nanovllm_amd.kernels.varlen import gather_kv, varlen_attention
from nanovllm_amd.layers.attention import Attention
from nanovllm_amd.utils.context import reset_context, set_context
from tests import fp4_oracle as fo

U8 = torch.uint8
BF = torch.bfloat16


def _i32(*v):
    return torch.tensor(v, dtype=torch.int32)


def _pool(blocks=4, page=32, kvh=2, **kw):
    p = dict(k_cache=torch.zeros(blocks, page, kvh, 64, dtype=U8),
             v_cache=torch.zeros(blocks, page, kvh, 64, dtype=U8),
             k_scale=torch.zeros(blocks, page, kvh, 4, dtype=U8),
             v_scale=torch.zeros(blocks, page, kvh, 4, dtype=U8))
    p.update(kw)
    return p


BAD_POOLS = [
    dict(k_scale=None), dict(v_scale=None), dict(k_cache=torch.zeros(4, 32, 2, 64)),
    dict(k_cache=torch.zeros(4, 32, 2, 128, dtype=U8)),
    dict(v_cache=torch.zeros(4, 32, 3, 64, dtype=U8)),
    dict(k_scale=torch.zeros(4, 32, 2, dtype=U8)), dict(v_scale=torch.zeros(4, 32, 2, 4)),
    dict(k_scale=torch.zeros(4, 32, 2, 8, dtype=U8)),
]


def _store(key=None, value=None, slots=None, **kw):
    key = torch.zeros(3, 2, 128, dtype=BF) if key is None else key
    return store_kvcache_fp4(key, key.clone() if value is None else value, **_pool(**kw),
                             slot_mapping=torch.zeros(3, dtype=torch.int32) if slots is None
                             else slots)


@pytest.mark.parametrize("bad", BAD_POOLS + [
    dict(key=torch.zeros(3, 2, 64, dtype=BF)), dict(key=torch.zeros(3, 3, 128, dtype=BF)),
    dict(key=torch.zeros(3, 2, 128)), dict(value=torch.zeros(2, 2, 128, dtype=BF)),
    dict(key=torch.zeros(3, 256, dtype=BF)),
])
def test_store_refuses(bad):
    with pytest.raises(ValueError):
        _store(**bad)


def test_store_layouts_and_device():
    with pytest.raises(AssertionError):
        _store(slots=torch.zeros(2, dtype=torch.int32))
    with pytest.raises(AssertionError):
        _store(key=torch.zeros(3, 128, 2, dtype=BF).transpose(1, 2))
    with pytest.raises(AssertionError):
        _store(k_cache=torch.zeros(4, 32, 2, 128, dtype=U8)[..., ::2])
    with pytest.raises(RuntimeError, match="device"):
        _store()


def _decode(q=None, tables=None, lens=None, out=None, fn=None, **kw):
    q = torch.zeros(3, 8, 128, dtype=BF) if q is None else q
    p = _pool(**kw)
    tables = torch.zeros(3, 1, dtype=torch.int32) if tables is None else tables
    lens = torch.ones(3, dtype=torch.int32) if lens is None else lens
    if fn is not None:
        return fn(q, p["k_cache"], p["v_cache"], tables, lens, 0.1, 32, k_scale=p["k_scale"],
                  v_scale=p["v_scale"])
    return paged_decode_fp4(q, p["k_cache"], p["v_cache"], p["k_scale"], p["v_scale"], tables,
                            lens, 0.1, out)


@pytest.mark.parametrize("bad", BAD_POOLS + [
    dict(q=torch.zeros(3, 8, 64, dtype=BF)), dict(q=torch.zeros(3, 9, 128, dtype=BF)),
    dict(q=torch.zeros(3, 8, 128)), dict(q=torch.zeros(8, 128, dtype=BF)), dict(page=48),
    dict(tables=torch.zeros(2, 1, dtype=torch.int32)), dict(tables=torch.zeros(3)),
    dict(lens=torch.ones(2, dtype=torch.int32)), dict(out=torch.zeros(3, 8, 128)),
    dict(out=torch.zeros(2, 8, 128, dtype=BF)),
    dict(out=torch.zeros(3, 8, 256, dtype=BF)[..., ::2]),
])
def test_decode_refuses(bad):
    with pytest.raises(ValueError):
        _decode(**bad)


def test_decode_needs_scales_and_device_tensors():
    with pytest.raises(ValueError, match="scale"):
        _decode(fn=lambda q, k, v, *a, **kw: paged_decode_attention(q, k, v, *a))
    for fn in (None, paged_decode_attention):
        with pytest.raises(RuntimeError, match="device"):
            _decode(fn=fn)
    p = _pool()
    with pytest.raises(RuntimeError, match="device"):
        paged_decode_append_fp4(torch.zeros(3, 8, 128, dtype=BF), torch.zeros(3, 2, 128, dtype=BF),
                                torch.zeros(3, 2, 128, dtype=BF), **p,
                                slot_mapping=torch.zeros(3, dtype=torch.int32),
                                block_tables=torch.zeros(3, 1, dtype=torch.int32),
                                context_lens=torch.ones(3, dtype=torch.int32), scale=0.1)


def test_dequant_and_gather_refuse():
    for codes, scale in ((torch.zeros(3, 64), torch.zeros(3, 4, dtype=U8)),
                         (torch.zeros(3, 32, dtype=U8), torch.zeros(3, 4, dtype=U8)),
                         (torch.zeros(3, 64, dtype=U8), torch.zeros(2, 4, dtype=U8)),
                         (torch.zeros(3, 64, dtype=U8), torch.zeros(3, 2, dtype=U8))):
        with pytest.raises(ValueError):
            dequant_fp4(codes, scale)
    with pytest.raises(RuntimeError, match="device"):
        dequant_fp4(torch.zeros(3, 64, dtype=U8), torch.zeros(3, 4, dtype=U8))
    p = _pool()
    args = (p["k_cache"], p["v_cache"])
    cu = torch.tensor([0, 5], dtype=torch.int32)
    with pytest.raises(ValueError, match="scale"):
        gather_kv(*args, torch.zeros(1, 1, dtype=torch.int32), cu, [0, 5])
    with pytest.raises(ValueError, match="rows"):
        gather_kv(*args, torch.zeros(1, 1, dtype=torch.int32), cu, [0, 5], block_table_row0=1,
                  k_scale=p["k_scale"], v_scale=p["v_scale"])
    with pytest.raises(RuntimeError, match="device"):
        gather_kv(*args, torch.zeros(1, 1, dtype=torch.int32), cu, [0, 5], k_scale=p["k_scale"],
                  v_scale=p["v_scale"])


def test_varlen_needs_scales():
    p = _pool()
    with pytest.raises(ValueError, match="scale"):
        varlen_attention(torch.zeros(3, 8, 128, dtype=BF), p["k_cache"], p["v_cache"], scale=0.1,
                         block_tables=torch.zeros(1, 1, dtype=torch.int32),
                         cu_seqlens_q_list=[0, 3], cu_seqlens_k_list=[0, 3])


@pytest.fixture
def recorded(monkeypatch):
    """Device calls recorded instead of made: what the checks let through, on the CPU."""
    calls = []
    monkeypatch.setattr(_native, "require_device", lambda *_: None)
    monkeypatch.setattr(_native, "stream_of", lambda *_: 0)
    monkeypatch.setattr(_native, "call_on", lambda t, name, *args: calls.append((name, args)))
    monkeypatch.setattr(_native, "call", lambda name, *args: calls.append((name, args)))
    return calls


def _append_call(**kw):
    p = _pool(**{n: kw.pop(n) for n in ("k_scale", "page") if n in kw})
    args = dict(q=torch.zeros(3, 8, 128, dtype=BF), key=torch.zeros(3, 2, 128, dtype=BF),
                value=torch.zeros(3, 2, 128, dtype=BF), slot_mapping=_i32(0, 1, 2),
                block_tables=torch.zeros(3, 1, dtype=torch.int32), context_lens=_i32(1, 1, 1))
    args.update(kw)
    return paged_decode_append_fp4(**args, **p, scale=0.1)


@pytest.mark.parametrize("bad", [
    dict(out=torch.zeros(3, 8, 128)), dict(out=torch.zeros(2, 8, 128, dtype=BF)),
    dict(q=torch.zeros(3, 7, 128, dtype=BF)), dict(q=torch.zeros(3, 8, 64, dtype=BF)),
    dict(q=torch.zeros(3, 8, 128)), dict(page=48), dict(k_scale=None),
    dict(block_tables=torch.zeros(2, 1, dtype=torch.int32)), dict(block_tables=_i32(0, 0, 0)),
    dict(context_lens=_i32(1, 1)), dict(slot_mapping=_i32(0)),
    dict(key=torch.zeros(3, 2, 64, dtype=BF)), dict(value=torch.zeros(3, 3, 128, dtype=BF)),
])
def test_append_and_attend_checks_all_before_it_stores(recorded, bad):
    with pytest.raises((ValueError, AssertionError)):
        _append_call(**bad)
    assert not recorded
    _append_call()
    assert [name for name, _ in recorded] == ["kvc_paged_decode_append_fp4"]


def _varlen(cu_q, cu_k, list_q, list_k, tables=1, decode=0, lens=None, width=1):
    p = _pool()
    q = torch.zeros(decode + list_q[-1], 8, 128, dtype=BF)
    varlen_attention(q, p["k_cache"], p["v_cache"], scale=0.1,
                     block_tables=torch.zeros(tables, width, dtype=torch.int32),
                     num_decode_rows=decode, decode_context_lens=lens, cu_seqlens_q=cu_q,
                     cu_seqlens_k=cu_k, cu_seqlens_q_list=list_q, cu_seqlens_k_list=list_k,
                     k_scale=p["k_scale"], v_scale=p["v_scale"])


def test_varlen_sequences_are_those_of_the_host_lists(recorded):
    """Offsets and lengths in tensors longer than the call's: what lies behind is not
    the call's, and needs no table rows."""
    long_q, long_k = _i32(0, 3, 5, 9), _i32(0, 20, 31, 40)
    _varlen(long_q, long_k, [0, 3], [0, 20])
    (name, args), = recorded
    assert name == "kvc_varlen_fp4" and args[18] == 1
    recorded.clear()
    _varlen(long_q, long_k, [0, 3], [0, 20], tables=3, decode=2, lens=_i32(4, 5, 6, 7))
    (name, args), = recorded
    assert name == "kvc_varlen_fp4" and args[16] == 2 and args[18] == 1
    recorded.clear()
    # decode rows alone
    _varlen(long_q, long_k, [0], [0], tables=2, decode=2, lens=_i32(4, 5, 6, 7))
    (name, args), = recorded
    assert name == "kvc_paged_decode_fp4"


@pytest.mark.parametrize("kw", [
    dict(cu_q=_i32(0, 3)), dict(cu_k=_i32(0, 20)), dict(cu_k=_i32()), dict(lens=_i32(4)),
])
def test_varlen_refuses_short_offsets_and_lengths(recorded, kw):
    args = dict(cu_q=_i32(0, 3, 5), cu_k=_i32(0, 20, 31), list_q=[0, 3, 5], list_k=[0, 20, 31],
                tables=4, decode=2, lens=_i32(4, 5))
    _varlen(**args)
    assert len(recorded) == 1
    recorded.clear()
    with pytest.raises(ValueError, match="fewer"):
        _varlen(**{**args, **kw})
    assert not recorded
    long = dict(list_q=[0, 500, 512], list_k=[0, 20000, 30000])       # gathered
    _varlen(**{**args, **long})
    assert [n for n, _ in recorded][:2] == ["kvc_paged_decode_fp4", "kvc_gather_kv_fp4"]
    recorded.clear()
    with pytest.raises(ValueError, match="fewer"):
        _varlen(**{**args, **long, **kw})
    assert not recorded


# --- the C entries ----------------------------------------------------------------

def _ptr(a):
    return a.ctypes.data


def test_c_entries_refuse_before_the_device():
    buf = np.zeros(4096, dtype=np.uint8)
    p = _ptr(buf) + (-_ptr(buf)) % 16
    lib = _native.load()

    def decode(page=32, kvh=2, dim=128, heads=8, blocks=4, max_blocks=1, batch=3, q=p, k=p, ks=p,
               lens=p, tables=p, ws=None, ws_bytes=0, stride=1024):
        return lib.kvc_paged_decode_fp4(q, stride, 128, k, p, ks, p, blocks, page, kvh, dim,
                                        tables, 1, max_blocks, lens, batch, heads,
                                        ctypes.c_float(0.1), p, stride, 128, ws, ws_bytes, None)

    assert decode(batch=0) == 0
    for bad in (dict(page=48), dict(page=0), dict(kvh=0), dict(dim=64), dict(heads=9),
                dict(blocks=-1), dict(max_blocks=-1), dict(max_blocks=1 << 22), dict(batch=-1),
                dict(q=None), dict(k=None), dict(ks=None), dict(lens=None), dict(tables=None),
                dict(batch=1 << 23, max_blocks=1 << 20)):
        assert decode(**bad) == -1, bad
    for bad in (dict(q=p + 8), dict(k=p + 4), dict(ks=p + 2), dict(stride=1028)):
        assert decode(**bad) == -2, bad
    need = lib.kvc_paged_decode_fp4_workspace_bytes(3, 8, 2, 32, 4096)
    assert need > 0
    assert decode(max_blocks=4096, ws=p, ws_bytes=need - 1) == -4
    assert decode(max_blocks=4096, ws=None, ws_bytes=need) == -4
    assert decode(max_blocks=4096, ws=p + 8, ws_bytes=need) == -2
    assert lib.kvc_paged_decode_fp4_workspace_bytes(3, 9, 2, 32, 4096) == 0

    def append(page=32, kvh=2, dim=128, heads=8, blocks=4, max_blocks=1, batch=3, n=3, q=p, k=p,
               key=p, slots=p, sb=4, lens=p, ws=None, ws_bytes=0, stride=1024, kstride=256):
        return lib.kvc_paged_decode_append_fp4(
            q, stride, 128, key, kstride, 128, p, kstride, 128, slots, sb, n, k, p, p, p, blocks,
            page, kvh, dim, p, 1, max_blocks, lens, batch, heads, ctypes.c_float(0.1), p, stride,
            128, ws, ws_bytes, None)

    assert append(batch=0, n=0) == 0
    for bad in (dict(page=48), dict(kvh=0), dict(dim=64), dict(heads=9), dict(blocks=-1),
                dict(max_blocks=1 << 22), dict(batch=-1), dict(n=-1), dict(sb=2), dict(q=None),
                dict(k=None), dict(key=None), dict(slots=None), dict(lens=None)):
        assert append(**bad) == -1, bad
    for bad in (dict(q=p + 8), dict(key=p + 2), dict(stride=1028), dict(kstride=260),
                dict(k=p + 4)):
        assert append(**bad) == -2, bad
    assert append(max_blocks=4096, ws=p, ws_bytes=need - 1) == -4

    def store(n=3, kvh=2, dim=128, sb=4, key=p, cache=p, slots=p, stride=256):
        return lib.kvc_store_fp4(key, stride, 128, p, stride, 128, cache, p, p, p, 128, slots, sb,
                                 n, kvh, dim, None)

    assert store(n=0) == 0
    for bad in (dict(dim=64), dict(kvh=0), dict(sb=2), dict(n=-1), dict(n=1 << 40),
                dict(key=None), dict(cache=None), dict(slots=None)):
        assert store(**bad) == -1, bad
    for bad in (dict(key=p + 2), dict(stride=260)):
        assert store(**bad) == -2, bad

    def gather(total=3, page=32, kvh=2, dim=128, chunks=1, cache=p, out=p, cu=p):
        return lib.kvc_gather_kv_fp4(cache, p, p, p, 4, page, kvh, dim, p, 1, 1, 0, chunks, cu,
                                     total, out, p, None)

    assert gather(total=0) == 0 and gather(chunks=0) == 0
    for bad in (dict(page=0), dict(kvh=0), dict(dim=64), dict(total=-1), dict(cache=None),
                dict(out=None), dict(cu=None), dict(total=1 << 40)):
        assert gather(**bad) == -1, bad
    assert gather(out=p + 8) == -2
    assert lib.kvc_dequant_fp4(p, p, 0, 128, p, None) == 0
    assert lib.kvc_dequant_fp4(p, p, 1, 64, p, None) == -1
    assert lib.kvc_dequant_fp4(None, p, 1, 128, p, None) == -1
    assert lib.kvc_dequant_fp4(p, p, 1, 128, p + 8, None) == -2

    def rows(tokens=5, decode=1, chunks=1, cu=p, blocks=0):
        return lib.kvc_varlen_fp4(p, 1024, 128, tokens, 8, p, p, p, p, 4, 32, 2, 128, p, 1, 1,
                                  decode, p, chunks, blocks, cu, cu, ctypes.c_float(0.1), p, 1024,
                                  128, None, 0, None)

    assert rows(tokens=0, decode=0, chunks=0) == 0
    for bad in (dict(decode=6), dict(decode=-1), dict(chunks=-1), dict(cu=None),
                dict(tokens=1 << 24)):
        assert rows(**bad) == -1, bad


def test_in_place_rule_is_host_only_and_monotone():
    def blocks(q, k, heads=32, kvh=4, table=1024, dec=0):
        cu_q, cu_k = (np.asarray(x, dtype=np.int32) for x in (q, k))
        return _native.query("kvc_varlen_fp4_blocks", _ptr(cu_q), _ptr(cu_k), len(q) - 1, heads,
                             kvh, 256, table, dec)

    assert blocks([0, 8], [0, 4096]) == 4              # 8 tokens x 8 heads, 16 columns a block
    assert blocks([0, 8, 8, 11], [0, 4096, 4096, 4500]) == 4 + 2
    assert blocks([0, 2048], [0, 16384]) == 0          # long chunks are gathered
    assert blocks([0, 0], [0, 5]) == 0 and blocks([0], [0]) == 0
    assert blocks([0, 8], [0, 4096], heads=9) == 0


# --- step tables ------------------------------------------------------------------

def _tables_args(batch=3, width=4, **kw):
    a = dict(context_lens=torch.zeros(batch, dtype=torch.int32),
             query_lens=torch.ones(batch, dtype=torch.int32),
             block_tables=torch.zeros(batch, width, dtype=torch.int32),
             num_blocks=torch.zeros(batch, dtype=torch.int32),
             free_blocks=torch.arange(8, dtype=torch.int32), num_free=_i32(8), page_size=32,
             max_tokens=8)
    a.update(kw)
    return a


@pytest.mark.parametrize("bad", [
    dict(block_tables=torch.zeros(3, 4)), dict(block_tables=torch.zeros(3, dtype=torch.int32)),
    dict(block_tables=torch.zeros(4, 3, dtype=torch.int32).t()),
    dict(block_tables=torch.zeros(1, 4, dtype=torch.int32).expand(3, 4)),
    dict(context_lens=_i32(1, 2)), dict(context_lens=torch.zeros(3)), dict(query_lens=_i32(1)),
    dict(num_blocks=torch.zeros(3, dtype=torch.int64)), dict(num_free=_i32(1, 2)),
    dict(free_blocks=torch.zeros(8)), dict(page_size=0), dict(max_tokens=-1),
    dict(tokens_per_row=2, max_tokens=7), dict(tokens_per_row=-1), dict(pad_slot=2 ** 31),
    dict(finished=torch.zeros(3)), dict(finished=torch.zeros(2, dtype=torch.bool)),
    dict(out=new_step_tables(3, 7, "cpu")), dict(out=new_step_tables(2, 8, "cpu")),
])
def test_step_tables_refuse(bad):
    with pytest.raises(ValueError):
        build_step_tables(**_tables_args(**bad))


def test_step_tables_refuse_rows_in_one_place():
    """Tables of one page a row, all rows over the same entry."""
    shared = torch.zeros(1, 1, dtype=torch.int32)
    with pytest.raises(ValueError, match="overlapping"):
        build_step_tables(**_tables_args(width=1, block_tables=shared.expand(3, 1)))
    with pytest.raises(ValueError, match="overlapping"):
        build_step_tables(**_tables_args(block_tables=torch.zeros(7, dtype=torch.int32).as_strided(
            (3, 4), (1, 1))))
    for fine in (torch.zeros(3, 1, dtype=torch.int32), torch.zeros(3, 0, dtype=torch.int32),
                 torch.zeros(3, 2, dtype=torch.int32)[:, :1],
                 torch.zeros(1, 4, dtype=torch.int32).expand(1, 4)):
        args = _tables_args(batch=fine.size(0), block_tables=fine)
        with pytest.raises(RuntimeError, match="device"):
            build_step_tables(**args)


def test_step_tables_need_device_tensors():
    for kw in ({}, dict(out=new_step_tables(3, 8, "cpu"))):
        with pytest.raises(RuntimeError, match="device"):
            build_step_tables(**_tables_args(**kw))


def test_c_step_tables_refuse():
    lib = _native.load()
    bufs = [np.zeros(64, dtype=np.int64) for _ in range(16)]
    p = [_ptr(b) for b in bufs]

    def call(batch=2, width=2, page=32, tokens=4, per_row=0, free=4, lens=p[0], query_out=p[7],
             seq_out=p[8], num=p[5], slots=p[10], cu_k=p[15]):
        return lib.kvc_step_tables(lens, p[1], None, p[2], width, width, batch, p[3], p[4], free,
                                   num, page, tokens, per_row, 0, slots, p[11], query_out, seq_out,
                                   p[9], p[12], p[13], p[14], cu_k, None)

    for bad in (dict(batch=-1), dict(batch=1 << 20), dict(width=-1), dict(width=1 << 29),
                dict(page=0), dict(page=1 << 21), dict(tokens=-1), dict(tokens=1 << 24),
                dict(per_row=3), dict(per_row=-1), dict(free=-1), dict(lens=None),
                dict(num=None), dict(slots=None), dict(query_out=p[0]), dict(seq_out=p[0]),
                dict(seq_out=p[1]), dict(seq_out=p[7]), dict(cu_k=p[14]), dict(slots=p[2]),
                dict(query_out=p[3])):
        assert call(**bad) == -1, bad


def test_c_step_tables_ended_refuse():
    """The lengths of ended rows go over context_lens or a place of their own."""
    lib = _native.load()
    bufs = [np.zeros(64, dtype=np.int64) for _ in range(17)]
    p = [_ptr(b) for b in bufs]

    def call(ended):
        return lib.kvc_step_tables_ended(p[0], p[1], p[6], ended, p[2], 2, 2, 2, p[3], p[4], 4,
                                         p[5], 32, 4, 0, 0, p[10], p[11], p[7], p[8], p[9], p[12],
                                         p[13], p[14], p[15], None)

    for i in list(range(1, 16)):
        assert call(p[i]) == -1, i
        assert b"ended_lens" in lib.kvc_last_error()


def test_device_tables_refuse():
    for bad in ((0, 4, 32, 8), (3, 0, 32, 8), (3, 4, 0, 8), (3, 4, 32, [1, 1]), (3, 4, 32, [-1]),
                (3, 4, 256, [1 << 23])):
        with pytest.raises(ValueError):
            DeviceBlockTables(*bad, device="cpu")
    t = DeviceBlockTables(3, 4, 32, 8, device="cpu")
    ones = torch.ones(3, dtype=torch.int32)
    for out, advance in ((new_step_tables(3, 3, "cpu"), True), (t.outputs(3), False),
                         (t.outputs(3, False), True),
                         (DeviceBlockTables(3, 4, 32, 8, device="cpu").outputs(3), True)):
        with pytest.raises(ValueError, match="outputs"):
            t.step(ones, 3, advance=advance, out=out)
    with pytest.raises(RuntimeError, match="device"):
        t.step(ones, 3)


# --- layers and runners -------------------------------------------------------------

def test_runner_arguments():
    for bad in (dict(kv_int8="tokhead"), dict(head_dim=64)):
        with pytest.raises(ValueError):
            KVCacheRunner(**{**dict(num_layers=1, num_blocks=2, block_size=32, num_kv_heads=2,
                                    head_dim=128, kv_fp4=True, device="cpu"), **bad})
    with pytest.raises(AssertionError):
        KVCacheRunner(1, 2, 32, 2, 128, kv_fp4=True, device="cpu", kv_offload_host_blocks=1)


def test_runner_tables_are_of_its_blocks():
    """Blocks behind the pool, the padding's scratch block among them, are refused:
    appends there would be dropped or shared."""
    runner = KVCacheRunner.__new__(KVCacheRunner)     # (the whole of it needs a GPU)
    runner.kv_cache = torch.zeros(2, 1, 7, 32, 2, 64, dtype=U8)
    runner.num_kvcache_blocks, runner.block_size, runner.scratch_slot = 6, 32, 6 * 32
    assert runner.device_tables(2, 3).num_free.tolist() == [6]
    assert runner.device_tables(2, 3, 4).free_blocks.tolist() == [0, 1, 2, 3]
    assert runner.device_tables(2, 3, torch.tensor([5, 2])).free_blocks.tolist() == [5, 2]
    assert runner.device_tables(2, 3, []).num_free.tolist() == [0]
    for bad in (7, [6], [0, 9], torch.tensor([6]), range(7)):
        with pytest.raises(ValueError, match="blocks"):
            runner.device_tables(2, 3, bad)


def test_decode_from_tables_of_another_page_size():
    """Slots and pages counted in other pages would be those of other tokens."""
    runner = KVCacheRunner.__new__(KVCacheRunner)
    runner.kv_cache, runner.block_size = torch.zeros(2, 1, 7, 32, 2, 64, dtype=U8), 32
    with pytest.raises(ValueError, match="pages of 64"):
        runner.prepare_decode_device(DeviceBlockTables(2, 3, 64, 6, device="cpu"))
    with pytest.raises(ValueError, match="meta"):
        runner.prepare_decode_device(DeviceBlockTables(2, 3, 32, 6, device="meta"))
    with pytest.raises(RuntimeError, match="device"):
        runner.prepare_decode_device(DeviceBlockTables(2, 3, 32, 6, device="cpu"))


def test_graph_runner_needs_scales_and_plain_scores():
    p = _pool()
    with pytest.raises(ValueError, match="scale"):
        DecodeGraphRunner([p["k_cache"]], [p["v_cache"]], 8, 1, 1, 0.1)
    with pytest.raises(ValueError, match="bf16"):
        DecodeGraphRunner([p["k_cache"]], [p["v_cache"]], 8, 1, 1, 0.1,
                          k_scales=[p["k_scale"]], v_scales=[p["v_scale"]],
                          score_shapes=dict(softcap=20.0))


def test_shaped_layers_refuse_a_4_bit_pool():
    layer = Attention(8, 128, 0.1, 2, softcap=30.0)
    p = _pool()
    layer.k_cache, layer.v_cache = p["k_cache"], p["v_cache"]
    layer.k_scale, layer.v_scale = p["k_scale"], p["v_scale"]
    set_context(False, slot_mapping=_i32(0), context_lens=_i32(1),
                block_tables=torch.zeros(1, 1, dtype=torch.int32))
    try:
        with pytest.raises(ValueError, match="bf16 pool"):
            layer(torch.zeros(1, 8 * 128, dtype=BF), torch.zeros(1, 256, dtype=BF),
                  torch.zeros(1, 256, dtype=BF))
    finally:
        reset_context()


# --- the oracle ---------------------------------------------------------------------

def test_oracle_encoding_by_hand():
    x = torch.zeros(1, 128)
    x[0, :9] = torch.tensor([6.0, -5.0, 5.5, 0.25, -0.75, 1.75, 2.5, 3.5, 0.2])
    x[0, 32] = 6.5                      # over 6: the next power, 3.25 rounds to 3
    x[0, 64] = float("inf")
    x[0, 96] = 2.0 ** -130
    codes, powers = fo.encode(x)
    assert powers.tolist() == [[127, 128, 255, 1]]
    got = fo.values(codes, powers)[0]
    assert got[:9].tolist() == [6.0, -4.0, 6.0, 0.0, -1.0, 2.0, 2.0, 4.0, 0.0]
    assert got[32] == 6.0 and torch.isnan(got[64:96]).all() and got[96] == 0
    assert codes[0, 0] == 7 + 16 * (8 + 6) and not codes[0, 32:48].any()
    big, power = fo.encode(torch.full((128,), 3.3e38))
    assert power.tolist() == [252] * 4 and torch.isfinite(fo.values(big, power)).all()
