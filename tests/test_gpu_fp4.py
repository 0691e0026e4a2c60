"""The 4-bit KV pool's kernels against the 64-bit oracle: append, dequantising reads,
paged decode, chunks read in place and chunks gathered."""
import math

import numpy as np
import pytest
import torch

from nanovllm_amd import _native
from nanovllm_amd.kernels.kv_fp4 import (dequant_fp4, paged_decode_append_fp4, paged_decode_fp4,
                                         store_kvcache_fp4, varlen_fp4)
from nanovllm_amd.kernels.paged_attention import paged_decode_attention
from nanovllm_amd.kernels.varlen import gather_kv, varlen_attention
from tests import fp4_oracle as fo
from tests import scored_oracle as so

pytestmark = pytest.mark.gpu
BF = torch.bfloat16
U8 = torch.uint8
SCALE = 128 ** -0.5


def _dev(pool):
    return tuple(t.cuda() for t in pool)


def _empty(blocks, page, kvh, fill=0x5a):
    return tuple(torch.full((blocks, page, kvh, w), fill, dtype=U8, device="cuda")
                 for w in (64, 64, 4, 4))


# --- append and reads ----------------------------------------------------------------

def test_append_every_bf16_value():
    """All 65536 bf16 values, among neighbours and among strangers: codes and powers
    equal the oracle's."""
    every = torch.arange(65536, dtype=torch.int32).to(torch.int16).view(BF).view(512, 128)
    gen = torch.Generator().manual_seed(3)
    mixed = every.flatten()[torch.randperm(65536, generator=gen)].view(512, 128)
    fine = every[torch.isfinite(every.float()).all(1)]
    spread = fine.flatten()[torch.randperm(fine.numel(), generator=gen)].view(-1, 128)
    rows = torch.cat((every, mixed, spread))[:, None].contiguous()
    n = rows.size(0)
    want, powers = fo.encode(rows)
    k, v, ks, vs = _empty((n + 31) // 32, 32, 1)
    key = rows.cuda()
    store_kvcache_fp4(key, key.flip(0), k, v, ks, vs, torch.arange(n, device="cuda"))
    torch.cuda.synchronize()
    assert torch.equal(ks.view(-1, 1, 4)[:n].cpu(), powers)
    assert torch.equal(vs.view(-1, 1, 4)[:n].cpu(), powers.flip(0))
    # a finite run's codes; a NaN run's are 0
    assert torch.equal(k.view(-1, 1, 64)[:n].cpu(), want)
    assert torch.equal(v.view(-1, 1, 64)[:n].cpu(), want.flip(0))
    got = dequant_fp4(k.view(-1, 1, 64)[:n], ks.view(-1, 1, 4)[:n]).cpu()
    exact = fo.values(want, powers).to(BF)
    assert torch.equal(torch.isnan(got), torch.isnan(exact))
    assert torch.equal(got.nan_to_num(0.0), exact.nan_to_num(0.0))


@pytest.mark.parametrize("kvh", [1, 2, 3, 4, 8])
@pytest.mark.parametrize("n,index", [(1, torch.int64), (5, torch.int32), (77, torch.int64),
                                     (1000, torch.int32)])
def test_append_slots_and_strides(kvh, n, index):
    """Strided rows, negative slots and slots outside the pool, every byte of the pool
    compared."""
    gen = torch.Generator().manual_seed(n * 10 + kvh)
    blocks, page = n // 32 + 3, 32
    slots = torch.randperm(blocks * page, generator=gen)[:n].to(index)
    if n > 3:
        slots[1] -= blocks * page           # counts from the end
        slots[2] = blocks * page            # outside: skipped
        slots[3] = -blocks * page - 1
    qkv = torch.randn(n, (4 + 2 * kvh) * 128, generator=gen).to(BF).cuda()
    key = qkv[:, 4 * 128:(4 + kvh) * 128].view(n, kvh, 128)
    value = qkv[:, (4 + kvh) * 128:].view(n, kvh, 128)
    pool = _empty(blocks, page, kvh)
    want = [t.clone().flatten(0, 1) for t in pool]
    for i, x in enumerate((key, value)):
        codes, powers = fo.encode(x)
        for j, s in enumerate(slots.tolist()):
            s += blocks * page if s < 0 else 0
            if 0 <= s < blocks * page:
                want[i][s], want[2 + i][s] = codes[j].cuda(), powers[j].cuda()
    store_kvcache_fp4(key, value, *pool, slots.cuda())
    for got, w in zip(pool, want):
        assert torch.equal(got.flatten(0, 1), w)


def test_append_of_nothing_and_unaligned_rows():
    pool = _empty(2, 32, 2)
    before = [t.clone() for t in pool]
    store_kvcache_fp4(torch.zeros(0, 2, 128, dtype=BF, device="cuda"),
                      torch.zeros(0, 2, 128, dtype=BF, device="cuda"), *pool,
                      torch.zeros(0, dtype=torch.int32, device="cuda"))
    odd = torch.zeros(3 * 256 + 4, dtype=BF, device="cuda")[4:].view(3, 2, 128)
    with pytest.raises(AssertionError, match="aligned"):
        store_kvcache_fp4(odd, odd, *pool, torch.zeros(3, dtype=torch.int32, device="cuda"))
    assert all(torch.equal(a, b) for a, b in zip(pool, before))
    assert dequant_fp4(pool[0][:0], pool[2][:0]).shape == (0, 32, 2, 128)


@pytest.mark.parametrize("page,kvh,lens,row0", [(32, 4, [1, 33, 64, 0, 100], 0),
                                                (256, 8, [255, 256, 257], 2), (48, 3, [97, 5], 1)])
def test_gather(page, kvh, lens, row0):
    pool, tables, k, v = fo.paged([3] * row0 + lens, page, kvh, seed=page + kvh)
    cu = [0]
    for n in lens:
        cu.append(cu[-1] + n)
    kc, vc, ks, vs = _dev(pool)
    got = gather_kv(kc, vc, tables.cuda(), torch.tensor(cu, device="cuda"), cu,
                    block_table_row0=row0, k_scale=ks, v_scale=vs)
    for g, seqs in zip(got, (k, v)):
        assert torch.equal(g.cpu(), torch.cat(seqs[row0:]).to(BF))


def test_gather_index_types_strides_and_both_paths(monkeypatch):
    lens = [70, 1, 200]
    pool, tables, k, v = fo.paged([3] + lens, 32, 4, seed=51)
    cu = [0, 70, 71, 271]
    scales = dict(zip(("k_scale", "v_scale"), _dev(pool)[2:]))
    kc, vc = _dev(pool)[:2]
    wide = torch.full((tables.size(0), 2 * tables.size(1)), -5, dtype=torch.int32)
    wide[:, ::2] = tables
    forms = [(tables.cuda(), torch.int32), (tables.cuda().long(), torch.int64),
             (wide.cuda()[:, ::2], torch.int32)]
    for path in range(2):
        for bt, kind in forms:
            got = gather_kv(kc, vc, bt, torch.tensor(cu, dtype=kind, device="cuda"), cu,
                            block_table_row0=1, **scales)
            for g, seqs in zip(got, (k, v)):
                assert torch.equal(g.cpu(), torch.cat(seqs[1:]).to(BF)), (path, kind)
        assert gather_kv(kc, vc, forms[0][0], torch.zeros(1, dtype=torch.int32, device="cuda"),
                         [0], **scales)[0].shape == (0, 4, 128)
        monkeypatch.setattr(_native, "_host", _native._NoHostPath)
    with pytest.raises(ValueError, match="cu_seqlens_k"):
        gather_kv(kc, vc, forms[0][0], torch.zeros(2, dtype=torch.int32, device="cuda"), cu,
                  **scales)


def test_gather_of_bad_pages_is_zero():
    pool, tables, k, _ = fo.paged([96, 40], 32, 2, seed=5)
    tables[0, 1], tables[1, 0] = 1 << 20, -7
    cu = [0, 96, 136]
    kc, vc, ks, vs = _dev(pool)
    got, _ = gather_kv(kc, vc, tables.cuda(), torch.tensor(cu, device="cuda"), cu, k_scale=ks,
                       v_scale=vs)
    got = got.cpu()
    want = torch.cat(k).to(BF)
    want[32:64] = 0
    want[96:128] = 0
    assert torch.equal(got, want)


# --- decode -----------------------------------------------------------------------------

def _decode(pool, tables, lens, q, scale=SCALE, width=None, **kw):
    """Both ways to cut the work: the table as it is, and one wide enough that the
    call has to expect long rows."""
    kc, vc, ks, vs = _dev(pool)
    outs = []
    for cols in (tables.size(1), width or tables.size(1) + (1 << 16) // kc.size(1)):
        t = torch.full((tables.size(0), cols), -1, dtype=torch.int32)
        t[:, :tables.size(1)] = tables
        outs.append(paged_decode_fp4(q.cuda(), kc, vc, ks, vs, t.cuda(),
                                     torch.tensor(lens, dtype=torch.int32).cuda(), scale, **kw))
    return outs


def _expect(q, k, v, lens, scale=SCALE):
    out, bound = [], []
    for i, n in enumerate(lens):
        o, b = fo.attend(q[i:i + 1], k[i][:max(n, 0)], v[i][:max(n, 0)],
                         torch.ones(1, max(n, 0), dtype=torch.bool), scale)
        out.append(o)
        bound.append(b)
    return torch.cat(out), torch.cat(bound)


@pytest.mark.parametrize("heads,kvh", [(8, 1), (4, 4), (16, 2), (32, 4), (16, 8), (6, 3),
                                       (40, 2), (17, 1), (128, 4), (96, 6)])
@pytest.mark.parametrize("page", [32, 96, 256])
def test_decode_lengths(heads, kvh, page):
    lens = [0, 1, 31, 32, 33, 63, 64, 65, 127, 129, 300, 513, 700]
    pool, tables, k, v = fo.paged(lens, page, kvh, seed=heads + page)
    gen = torch.Generator().manual_seed(heads)
    q = torch.randn(len(lens), heads, 128, generator=gen).to(BF)
    want, bound = _expect(q, k, v, lens)
    for i, got in enumerate(_decode(pool, tables, lens, q)):
        fo.check(got, want, bound, f"{heads}/{kvh} page {page} {('short', 'wide')[i]} table")
        assert not got[0].any()                      # no keys: zeros


@pytest.mark.parametrize("batch,lo,hi,heads,kvh", [(1, 5000, 5000, 32, 4), (3, 900, 9000, 16, 8),
                                                   (70, 1, 400, 16, 2), (131, 64, 64, 8, 2),
                                                   (2, 20000, 33000, 8, 4), (64, 2048, 2048, 8, 4),
                                                   (300, 40, 100, 4, 2)])
def test_decode_batches(batch, lo, hi, heads, kvh):
    """Shares that hold many rows, rows that span many shares, equal rows, over 64 and
    over 256 rows."""
    gen = torch.Generator().manual_seed(batch)
    lens = torch.randint(lo, hi + 1, (batch,), generator=gen).tolist()
    pool, tables, k, v = fo.paged(lens, 256, kvh, seed=batch)
    q = torch.randn(batch, heads, 128, generator=gen).to(BF)
    want, bound = _expect(q, k, v, lens)
    for i, got in enumerate(_decode(pool, tables, lens, q)):
        fo.check(got, want, bound, f"batch {batch} {lo}..{hi} {i}")


@pytest.mark.parametrize("rows,heads,kvh,lo,hi", [(200, 8, 4, 1, 90), (300, 4, 4, 0, 300),
                                                  (90, 16, 8, 40, 40), (210, 16, 8, 1, 200),
                                                  (150, 48, 16, 1, 70), (260, 24, 2, 5, 40)])
def test_decode_many_short_rows(rows, heads, kvh, lo, hi):
    """Batches whose workgroups take several kv heads of a row whole."""
    gen = torch.Generator().manual_seed(rows)
    lens = torch.randint(lo, hi + 1, (rows,), generator=gen).tolist()
    pool, tables, k, v = fo.paged(lens, 32, kvh, seed=rows + kvh)
    q = torch.randn(rows, heads, 128, generator=gen).to(BF)
    got = paged_decode_fp4(q.cuda(), *_dev(pool), tables.cuda(),
                           torch.tensor(lens, dtype=torch.int32).cuda(), SCALE)
    want, bound = _expect(q, k, v, lens)
    fo.check(got, want, bound, f"{rows} rows of {lo} to {hi}")


@pytest.mark.parametrize("count,kvh", [(100, 8), (210, 8), (220, 4)])
def test_many_short_chunks_in_place(count, kvh):
    """The same of chunks, decode rows among them."""
    gen = torch.Generator().manual_seed(count)
    chunks = [(int(n), int(n + m)) for n, m in zip(
        torch.randint(0, 9, (count,), generator=gen), torch.randint(0, 60, (count,), generator=gen))]
    decode = torch.randint(0, 60, (20,), generator=gen).tolist()
    pool, tables, k, v = fo.paged(decode + [m for _, m in chunks], 32, kvh, seed=count + 1)
    q = torch.randn(20 + sum(n for n, _ in chunks), 2 * kvh, 128, generator=gen).to(BF)
    want, bound = _chunk_expect(q, k, v, decode, chunks)
    got = _chunk_call(pool, tables, decode, chunks, q, "known")
    fo.check(got, want, bound, f"{count} chunks")


@pytest.mark.parametrize("scale", [0.0, -SCALE, 1.0, 1e-20])
def test_decode_scales(scale):
    lens = [70, 200]
    pool, tables, k, v = fo.paged(lens, 32, 2, seed=9)
    gen = torch.Generator().manual_seed(1)
    q = torch.randn(2, 8, 128, generator=gen).to(BF)
    want, bound = _expect(q, k, v, lens, scale)
    for got in _decode(pool, tables, lens, q, scale):
        fo.check(got, want, bound, f"scale {scale}")


def test_decode_query_magnitudes():
    """Query elements over 40 binades, rows of zeros, tiny and large rows."""
    lens = [150] * 6
    pool, tables, k, v = fo.paged(lens, 32, 2, seed=10)
    gen = torch.Generator().manual_seed(2)
    q = torch.randn(6, 8, 128, generator=gen)
    q[0] *= 2.0 ** torch.randint(-40, 1, (8, 128), generator=gen).float()
    q[1] = 0
    q[2] *= 1e-30
    q[3] *= 40
    q[4, :, ::2] = 0
    q[5, :, 5] *= 300                       # one dim far wider than the others
    q = q.to(BF)
    want, bound = _expect(q, k, v, lens)
    for got in _decode(pool, tables, lens, q):
        fo.check(got, want, bound, "query magnitudes")


@pytest.mark.parametrize("size", [2.0 ** -100, 2.0 ** -20, 2.0 ** 30, 2.0 ** 100])
def test_decode_value_magnitudes(size):
    """V's powers over the format's range (K's stay near 1); runs of one row apart."""
    lens = [90, 64]
    pool, tables, k, _ = fo.paged(lens, 32, 2, seed=11)
    gen = torch.Generator().manual_seed(4)
    kc, vc, ks, vs = pool
    v = []
    for i, n in enumerate(lens):
        x = torch.randn(n, 2, 128, generator=gen) * size
        x[..., 32:64] *= 2.0 ** 10
        codes, powers = fo.encode(x.to(BF))
        pos = torch.arange(n)
        slot = tables[i, pos // 32].long() * 32 + pos % 32
        vc.flatten(0, 1)[slot], vs.flatten(0, 1)[slot] = codes, powers
        v.append(fo.values(codes, powers))
    q = torch.randn(2, 4, 128, generator=gen).to(BF)
    want, bound = _expect(q, k, v, lens)
    for got in _decode((kc, vc, ks, vs), tables, lens, q):
        fo.check(got, want, bound, f"values of {size}")


def test_decode_nan_and_infinite_inputs():
    """A NaN run of K makes its rows NaN; one of V its channels; a query with an
    infinity or a NaN its head; other rows stay as they are."""
    lens = [100, 100, 100, 40]
    pool, tables, k, v = fo.paged(lens, 32, 2, seed=12)
    gen = torch.Generator().manual_seed(5)
    q = torch.randn(4, 8, 128, generator=gen).to(BF)
    kc, vc, ks, vs = pool
    at = int(tables[0, 70 // 32]) * 32 + 70 % 32
    ks.flatten(0, 1)[at, 1, 2] = 255                 # row 0, kv head 1
    kc.flatten(0, 1)[at, 1, 32:48] = 0
    at = int(tables[1, 99 // 32]) * 32 + 99 % 32
    vs.flatten(0, 1)[at, 0, 1] = 255                 # row 1, kv head 0, channels 32 .. 63
    vc.flatten(0, 1)[at, 0, 16:32] = 0
    q[2, 3, 17] = float("inf")
    q[2, 6, 5] = float("nan")
    want, bound = _expect(q, k, v, lens)
    want[0, 4:] = math.nan
    want[1, :4, 32:64] = math.nan
    want[2, [3, 6]] = math.nan
    for got in _decode((kc, vc, ks, vs), tables, lens, q):
        fo.check(got, want, bound, "NaN runs")


def test_decode_lengths_and_tables_that_do_not_fit():
    """A length past its table counts the table's keys; negative lengths none; a bad
    table entry reads as zeros."""
    lens = [64, 64, 64]
    pool, tables, k, v = fo.paged(lens, 32, 2, seed=13)
    gen = torch.Generator().manual_seed(6)
    q = torch.randn(3, 4, 128, generator=gen).to(BF)
    want, bound = _expect(q, k, v, [64, 0, 64])
    kc, vc, ks, vs = _dev(pool)
    got = paged_decode_fp4(q.cuda(), kc, vc, ks, vs, tables.cuda(),
                           torch.tensor([1000, -5, 64], dtype=torch.int32).cuda(), SCALE)
    fo.check(got, want, bound, "lengths")
    bad = tables.clone()
    bad[0, 1], bad[2, 0] = 1 << 24, -1
    for i, rows in ((0, slice(32, 64)), (2, slice(0, 32))):
        k[i], v[i] = k[i].clone(), v[i].clone()
        k[i][rows], v[i][rows] = 0, 0
    want, bound = _expect(q, k, v, lens)
    for got in _decode(pool, bad, lens, q):
        fo.check(got, want, bound, "bad pages")


def test_decode_strides_and_given_output():
    lens = [90, 10, 33]
    pool, tables, k, v = fo.paged(lens, 32, 2, seed=14)
    gen = torch.Generator().manual_seed(7)
    wide = torch.randn(3, 12, 128, generator=gen).to(BF)
    q = wide[:, 2:10]
    want, bound = _expect(q, k, v, lens)
    kc, vc, ks, vs = _dev(pool)
    lens_t = torch.tensor(lens, device="cuda")             # int64
    tab = torch.full((5, 8), -1, dtype=torch.int64)
    tab[:3, 1:1 + tables.size(1)] = tables
    view = tab.cuda()[:, 1:1 + tables.size(1)]
    out = torch.full((3, 10, 128), 7.0, dtype=BF, device="cuda")
    got = paged_decode_fp4(wide.cuda()[:, 2:10], kc, vc, ks, vs, view, lens_t, SCALE,
                           out=out[:, 1:9])
    assert got.data_ptr() == out[:, 1:9].data_ptr()
    fo.check(got, want, bound, "given output")
    assert (out[:, 0] == 7).all() and (out[:, 9] == 7).all()
    odd = torch.zeros(3 * 8 * 128 + 1, dtype=BF, device="cuda")[1:].view(3, 8, 128)
    odd.copy_(q)
    fo.check(paged_decode_fp4(odd, kc, vc, ks, vs, view, lens_t, SCALE), want, bound, "odd q")
    fo.check(paged_decode_attention(q.cuda(), kc, vc, view, lens_t, SCALE, 90, k_scale=ks,
                                    v_scale=vs), want, bound, "paged_decode_attention")
    assert paged_decode_fp4(q[:0].cuda(), kc, vc, ks, vs, view[:0], lens_t[:0],
                            SCALE).shape == (0, 8, 128)


def test_decode_python_and_native_paths_agree(monkeypatch):
    lens = [500, 3]
    pool, tables, _, _ = fo.paged(lens, 32, 4, seed=15)
    q = torch.randn(2, 8, 128).to(BF).cuda()
    args = (*_dev(pool), tables.cuda(), torch.tensor(lens, dtype=torch.int32).cuda(), SCALE)
    key = torch.randn(2, 4, 128).to(BF).cuda()
    slots = torch.tensor([int(tables[0, 15]) * 32 + 19, int(tables[1, 0]) * 32 + 2],
                         dtype=torch.int32).cuda()
    first = paged_decode_fp4(q, *args)
    step = paged_decode_append_fp4(q, key, key, *args[:4], slots, *args[4:])
    stored = [t.clone() for t in args[:4]]
    monkeypatch.setattr(_native, "_host", _native._NoHostPath)
    for t, old in zip(args[:4], _dev(pool)):
        t.copy_(old)
    assert torch.equal(paged_decode_fp4(q, *args), first)
    assert torch.equal(paged_decode_append_fp4(q, key, key, *args[:4], slots, *args[4:]), step)
    assert all(torch.equal(a, b) for a, b in zip(args[:4], stored))


def test_decode_append():
    """The step's call: the new tokens are in the pool and attended."""
    lens = [1, 33, 64, 200]
    pool, tables, k, v = fo.paged(lens, 32, 2, seed=16)
    gen = torch.Generator().manual_seed(8)
    q = torch.randn(4, 8, 128, generator=gen).to(BF)
    key, value = (torch.randn(4, 2, 128, generator=gen).to(BF) for _ in range(2))
    slots = torch.tensor([int(tables[i, (n - 1) // 32]) * 32 + (n - 1) % 32
                          for i, n in enumerate(lens)])
    for seqs, x in ((k, key), (v, value)):
        new = fo.values(*fo.encode(x))
        for i, n in enumerate(lens):
            seqs[i] = torch.cat((seqs[i][:n - 1], new[i:i + 1]))
    want, bound = _expect(q, k, v, lens)
    dev = _dev(pool)
    got = paged_decode_append_fp4(q.cuda(), key.cuda(), value.cuda(), *dev, slots.cuda(),
                                  tables.cuda(), torch.tensor(lens, dtype=torch.int32).cuda(),
                                  SCALE)
    fo.check(got, want, bound, "append and attend")
    codes, powers = fo.encode(key)
    assert torch.equal(dev[0].flatten(0, 1)[slots.cuda()].cpu(), codes)
    assert torch.equal(dev[2].flatten(0, 1)[slots.cuda()].cpu(), powers)


def test_decode_over_pools_past_32_bits():
    """Blocks whose codes lie past 4 GiB, and whose rows pass 2^31 bytes of powers."""
    page, kvh = 256, 8
    blocks = (1 << 32) // (page * kvh * 64) + 6
    kc, vc = (torch.empty(blocks, page, kvh, 64, dtype=U8, device="cuda") for _ in range(2))
    ks, vs = (torch.empty(blocks, page, kvh, 4, dtype=U8, device="cuda") for _ in range(2))
    lens = [700, 300]
    pool, tables, k, v = fo.paged(lens, page, kvh, seed=17, spare=0)
    n = pool[0].size(0)
    for big, small in zip((kc, vc, ks, vs), pool):
        big[blocks - n:] = small.cuda()
    tables = torch.where(tables >= 0, tables + blocks - n, tables)
    q = torch.randn(2, 16, 128, generator=torch.Generator().manual_seed(9)).to(BF)
    want, bound = _expect(q, k, v, lens)
    got = paged_decode_fp4(q.cuda(), kc, vc, ks, vs, tables.cuda(),
                           torch.tensor(lens, dtype=torch.int32).cuda(), SCALE)
    fo.check(got, want, bound, "high blocks")
    wide = torch.full((2, 200), -1, dtype=torch.int32)
    wide[:, :tables.size(1)] = tables
    got = paged_decode_fp4(q.cuda(), kc, vc, ks, vs, wide.cuda(),
                           torch.tensor(lens, dtype=torch.int32).cuda(), SCALE)
    fo.check(got, want, bound, "high blocks, cut")
    got, _ = gather_kv(kc, vc, tables.cuda(), torch.tensor([0, 700], device="cuda"), [0, 700],
                       k_scale=ks, v_scale=vs)
    assert torch.equal(got.cpu(), k[0].to(BF))
    # (the last slot of the pool, which a sequence above may hold)
    slot = torch.tensor([blocks * page - 1], device="cuda")
    key = torch.randn(1, kvh, 128).to(BF)
    store_kvcache_fp4(key.cuda(), key.cuda(), kc, vc, ks, vs, slot)
    assert torch.equal(kc[-1, -1].cpu(), fo.encode(key)[0][0])


def test_decode_on_another_stream_and_in_two_at_once():
    lens = [3000, 40]
    pool, tables, k, v = fo.paged(lens, 32, 4, seed=18)
    gen = torch.Generator().manual_seed(10)
    qs = [torch.randn(2, 16, 128, generator=gen).to(BF) for _ in range(2)]
    args = (*_dev(pool), tables.cuda(), torch.tensor(lens, dtype=torch.int32).cuda(), SCALE)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    dq = [q.cuda() for q in qs]
    torch.cuda.synchronize()
    outs = [[], []]
    for _ in range(8):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                outs[i].append(paged_decode_fp4(dq[i], *args))
    torch.cuda.synchronize()
    for i in range(2):
        want, bound = _expect(qs[i], k, v, lens)
        for got in outs[i]:
            assert torch.equal(got, outs[i][0])
        fo.check(outs[i][0], want, bound, f"stream {i}")


@pytest.mark.parametrize("width", [4, 2200])
def test_decode_step_captured(width):
    """A captured step replayed for other lengths, tables, queries and tokens, with
    eager calls between; two graphs that share a memory pool."""
    page, kvh, heads, batch = 32, 4, 8, 3
    blocks = 40
    gen = torch.Generator().manual_seed(11)
    pool = _empty(blocks, page, kvh, 0)
    pool[2].fill_(127), pool[3].fill_(127)
    q = torch.zeros(batch, heads, 128, dtype=BF, device="cuda")
    key, value = (torch.zeros(batch, kvh, 128, dtype=BF, device="cuda") for _ in range(2))
    slots = torch.zeros(batch, dtype=torch.int32, device="cuda")
    tables = torch.full((batch, width), -1, dtype=torch.int32, device="cuda")
    lens = torch.ones(batch, dtype=torch.int32, device="cuda")
    tables[:, 0] = torch.tensor([0, 1, 2])
    slots.copy_(torch.tensor([0, 32, 64]))
    out = torch.zeros_like(q)

    def step():
        return paged_decode_append_fp4(q, key, value, *pool, slots, tables, lens, SCALE, out=out)

    step()
    torch.cuda.synchronize()
    graphs, shared = [], None
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, pool=shared):
            step()
        shared = g.pool()
        graphs.append(g)
    held = [t.clone() for t in pool]
    for t, h in zip(pool, held):
        t.copy_(h)
    k = [torch.zeros(0, kvh, 128, dtype=torch.float64) for _ in range(batch)]
    v = [x.clone() for x in k]
    order = torch.randperm(blocks, generator=gen)[:batch * 4].view(batch, 4)
    tables[:, :4] = order.to(torch.int32)
    for i in range(7):
        nk, nv = (torch.randn(batch, kvh, 128, generator=gen).to(BF) for _ in range(2))
        nq = torch.randn(batch, heads, 128, generator=gen).to(BF)
        pos = [len(x) for x in k]
        where = [int(order[b, pos[b] // page]) * page + pos[b] % page for b in range(batch)]
        q.copy_(nq), key.copy_(nk), value.copy_(nv)
        slots.copy_(torch.tensor(where))
        for b in range(batch):
            k[b] = torch.cat((k[b], fo.values(*fo.encode(nk))[b:b + 1]))
            v[b] = torch.cat((v[b], fo.values(*fo.encode(nv))[b:b + 1]))
        lens.copy_(torch.tensor([len(x) for x in k]))
        graphs[i % 2].replay()
        torch.cuda.synchronize()
        want, bound = _expect(nq, k, v, [len(x) for x in k])
        fo.check(out, want, bound, f"replay {i}")
        first = out.clone()
        assert torch.equal(step(), first)              # eager, between the replays
    # row 0 grows by 60 tokens at once
    extra = torch.randn(60, kvh, 128, generator=gen).to(BF)
    at = torch.tensor([int(order[0, (7 + j) // page]) * page + (7 + j) % page for j in range(60)])
    store_kvcache_fp4(extra.cuda(), extra.cuda(), *pool, at.cuda())
    k[0] = torch.cat((k[0], fo.values(*fo.encode(extra))))
    v[0] = torch.cat((v[0], fo.values(*fo.encode(extra))))
    lens[0] = 67
    for g in graphs:
        g.replay()
        torch.cuda.synchronize()
        want, bound = _expect(nq, k, v, [len(x) for x in k])
        fo.check(out, want, bound, "longer row")


# --- chunks ---------------------------------------------------------------------------------

def _chunk_call(pool, tables, decode, chunks, q, in_place, width=None, out=None):
    cu_q, cu_k = [0], [0]
    for n, m in chunks:
        cu_q.append(cu_q[-1] + n)
        cu_k.append(cu_k[-1] + m)
    kc, vc, ks, vs = _dev(pool)
    t = torch.full((tables.size(0), width or tables.size(1)), -1, dtype=torch.int32)
    t[:, :tables.size(1)] = tables
    dq, dk = (torch.tensor(x, dtype=torch.int32).cuda() for x in (cu_q, cu_k))
    lens = torch.tensor(decode, dtype=torch.int32).cuda()
    if in_place:
        group = q.size(1) // kc.size(2)
        blocks = sum((n * group + 15) // 16 for n, _ in chunks) if in_place == "known" else 0
        out = torch.empty_like(q.cuda()) if out is None else out
        return varlen_fp4(q.cuda(), kc, vc, ks, vs, t.cuda(), len(decode), lens, blocks, dq, dk,
                          SCALE, out)
    return varlen_attention(q.cuda(), kc, vc, scale=SCALE, block_tables=t.cuda(),
                            num_decode_rows=len(decode), decode_context_lens=lens,
                            cu_seqlens_q=dq, cu_seqlens_k=dk, cu_seqlens_q_list=cu_q,
                            cu_seqlens_k_list=cu_k, k_scale=ks, v_scale=vs,
                            decode_context_lens_list=decode)


def _chunk_expect(q, k, v, decode, chunks):
    out, bound, at = [], [], 0
    for i, (n, m) in enumerate([(1, m) for m in decode] + list(chunks)):
        o, b = fo.attend(q[at:at + n], k[i], v[i], fo.causal(n, m), SCALE)
        out.append(o)
        bound.append(b)
        at += n
    return torch.cat(out), torch.cat(bound)


@pytest.mark.parametrize("heads,kvh", [(16, 2), (16, 8), (3, 3), (40, 2), (8, 1)])
@pytest.mark.parametrize("decode,chunks", [
    ([], [(1, 1)]), ([], [(2, 65), (17, 17), (0, 0), (5, 700), (33, 64)]),
    ([40, 0, 513], [(3, 130), (0, 7), (9, 9)]), ([5], [(20, 2100)]), ([], [(65, 3000), (1, 31)])])
def test_chunks_read_in_place(heads, kvh, decode, chunks):
    lens = decode + [m for _, m in chunks]
    pool, tables, k, v = fo.paged(lens, 32, kvh, seed=heads + len(lens))
    gen = torch.Generator().manual_seed(len(lens))
    q = torch.randn(len(decode) + sum(n for n, _ in chunks), heads, 128, generator=gen).to(BF)
    want, bound = _chunk_expect(q, k, v, decode, chunks)
    for in_place, width in (("known", None), ("unknown", None), ("known", 2200)):
        got = _chunk_call(pool, tables, decode, chunks, q, in_place, width)
        fo.check(got, want, bound, f"{heads}/{kvh} {decode} {chunks} {in_place} {width}")


def test_many_chunks_in_place():
    """Over 64 sequences, most with more than one block."""
    gen = torch.Generator().manual_seed(19)
    chunks = [(int(n), int(n + m)) for n, m in zip(
        torch.randint(0, 12, (80,), generator=gen), torch.randint(0, 300, (80,), generator=gen))]
    decode = torch.randint(1, 400, (30,), generator=gen).tolist()
    pool, tables, k, v = fo.paged(decode + [m for _, m in chunks], 64, 2, seed=20)
    q = torch.randn(30 + sum(n for n, _ in chunks), 8, 128, generator=gen).to(BF)
    want, bound = _chunk_expect(q, k, v, decode, chunks)
    for width in (None, 1100):
        got = _chunk_call(pool, tables, decode, chunks, q, "known", width)
        fo.check(got, want, bound, f"110 sequences, width {width}")


@pytest.mark.parametrize("decode,chunks", [([], [(8, 4096)]), ([90, 700], [(70, 200), (300, 900)]),
                                           ([], [(513, 513)]), ([33], [])])
def test_varlen_attention(decode, chunks):
    """The public call, whichever way it reads the pool.  Gathered rows are bf16 and
    exact; the bf16 prefill's own roundings lie within the same bound as the in-place
    form's (a weight and the output in bf16)."""
    lens = decode + [m for _, m in chunks]
    pool, tables, k, v = fo.paged(lens, 256, 4, seed=21)
    gen = torch.Generator().manual_seed(12)
    q = torch.randn(len(decode) + sum(n for n, _ in chunks), 16, 128, generator=gen).to(BF)
    want, bound = _chunk_expect(q, k, v, decode, chunks)
    fo.check(_chunk_call(pool, tables, decode, chunks, q, False), want, bound, "varlen_attention")


def test_rows_of_no_sequence_stay():
    """Offsets that end before the last query row, and device lengths that disagree
    with the host's block count by being shorter."""
    pool, tables, k, v = fo.paged([64, 50], 32, 2, seed=22)
    gen = torch.Generator().manual_seed(13)
    q = torch.randn(12, 8, 128, generator=gen).to(BF)
    kc, vc, ks, vs = _dev(pool)
    for width in (2, 2200):
        t = torch.full((2, width), -1, dtype=torch.int32)
        t[:, :2] = tables
        out = torch.full((12, 8, 128), 3.0, dtype=BF, device="cuda")
        varlen_fp4(q.cuda(), kc, vc, ks, vs, t.cuda(), 0, None, 6,
                   torch.tensor([0, 4, 9], dtype=torch.int32).cuda(),
                   torch.tensor([0, 64, 114], dtype=torch.int32).cuda(), SCALE, out)
        want, bound = _chunk_expect(q[:9], k, v, [], [(4, 64), (5, 50)])
        fo.check(out[:9], want, bound, f"rows of sequences, width {width}")
        assert (out[9:] == 3).all()


def test_fewer_blocks_told_than_there_are():
    """The told blocks come first; what lies behind them is not joined, and nothing
    outside the output is written."""
    chunks = [(24, 90), (24, 120), (24, 64)]
    pool, tables, k, v = fo.paged([m for _, m in chunks], 32, 2, seed=24)
    gen = torch.Generator().manual_seed(14)
    q = torch.randn(72, 8, 128, generator=gen).to(BF)
    want, bound = _chunk_expect(q, k, v, [], chunks)
    kc, vc, ks, vs = _dev(pool)
    for width in (4, 2200):
        t = torch.full((3, width), -1, dtype=torch.int32)
        t[:, :4] = tables
        whole = torch.full((74, 8, 128), 3.0, dtype=BF, device="cuda")
        varlen_fp4(q.cuda(), kc, vc, ks, vs, t.cuda(), 0, None, 6,
                   torch.tensor([0, 24, 48, 72], dtype=torch.int32).cuda(),
                   torch.tensor([0, 90, 210, 274], dtype=torch.int32).cuda(), SCALE, whole[1:73])
        fo.check(whole[1:25], want[:24], bound[:24], f"told rows, width {width}")
        assert (whole[0] == 3).all() and (whole[73] == 3).all()


@pytest.mark.parametrize("decode,chunks,width", [
    ([300, 1, 40], [(4, 700), (9, 9)], 4), ([300, 1, 40], [(4, 700), (9, 9)], 200),
    ([64], [(300, 900)], 4)])
def test_chunks_captured(decode, chunks, width):
    """A mixed call in a graph, replayed over other pools, queries and decode lengths
    with eager calls between: each replay is the eager call's, bit for bit."""
    lens = decode + [m for _, m in chunks]
    pools = [fo.paged(lens, 256, 4, seed=60 + i, spare=2) for i in range(2)]
    kc, vc, ks, vs = state = _dev(pools[0][0])
    tables = torch.full((len(lens), width), -1, dtype=torch.int32, device="cuda")
    cu_q, cu_k = [0], [0]
    for n, m in chunks:
        cu_q.append(cu_q[-1] + n)
        cu_k.append(cu_k[-1] + m)
    dq, dk = (torch.tensor(x, dtype=torch.int32).cuda() for x in (cu_q, cu_k))
    held = torch.tensor(decode, dtype=torch.int32).cuda()
    gen = torch.Generator().manual_seed(15)
    q = torch.zeros(len(decode) + cu_q[-1], 16, 128, dtype=BF, device="cuda")

    def call():
        return varlen_attention(q, kc, vc, scale=SCALE, block_tables=tables,
                                num_decode_rows=len(decode), decode_context_lens=held,
                                cu_seqlens_q=dq, cu_seqlens_k=dk, cu_seqlens_q_list=cu_q,
                                cu_seqlens_k_list=cu_k, k_scale=ks, v_scale=vs,
                                decode_context_lens_list=decode)

    tables[:, :pools[0][1].size(1)] = pools[0][1].cuda()
    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    for i in range(6):
        pool, bt, k, v = pools[i % 2]
        for t, new in zip(state, pool):
            t.copy_(new)
        tables[:, :bt.size(1)] = bt.cuda()
        now = [max(0, n - 13 * i) for n in decode]
        held.copy_(torch.tensor(now))
        nq = torch.randn(q.shape, generator=gen).to(BF)
        q.copy_(nq)
        graph.replay()
        torch.cuda.synchronize()
        got = out.clone()
        assert torch.equal(call(), got), i
        if i % 3 == 1:
            short = [x[:n] for x, n in zip(k, now)] + k[len(now):]
            other = [x[:n] for x, n in zip(v, now)] + v[len(now):]
            fo.check(got, *_chunk_expect(nq, short, other, now, chunks), f"replay {i}")


def test_nan_runs_reach_only_the_tokens_that_see_them():
    chunks = [(6, 70)]
    pool, tables, k, v = fo.paged([70], 32, 2, seed=23)
    kc, vc, ks, vs = pool
    at = int(tables[0, 2]) * 32 + 67 - 64
    vs.flatten(0, 1)[at, 1, 3] = 255
    vc.flatten(0, 1)[at, 1, 48:] = 0
    q = torch.randn(6, 4, 128, generator=torch.Generator().manual_seed(14)).to(BF)
    want, bound = _chunk_expect(q, k, v, [], chunks)
    want[3:, 2:, 96:] = math.nan                    # tokens 64 + 3 .. see key 67
    for width in (None, 2200):
        got = _chunk_call((kc, vc, ks, vs), tables, [], chunks, q, "known", width)
        fo.check(got, want, bound, "NaN run of key 67")


def test_host_lists_absent_falls_back_to_python():
    pool, tables, k, v = fo.paged([40], 32, 2, seed=24)
    q = torch.randn(5, 8, 128, generator=torch.Generator().manual_seed(15)).to(BF)
    kc, vc, ks, vs = _dev(pool)
    got = varlen_attention(q.cuda(), kc, vc, scale=SCALE, block_tables=tables.cuda(),
                           cu_seqlens_q=torch.tensor([0, 5]).cuda(),
                           cu_seqlens_k=torch.tensor([0, 40]).cuda(), k_scale=ks, v_scale=vs)
    want, bound = _chunk_expect(q, k, v, [], [(5, 40)])
    fo.check(got, want, bound, "offsets on the device alone")


def test_bf16_pools_keep_their_path():
    """A bf16 decode beside a 4-bit one, and scales given for the wrong pool."""
    k_cache, v_cache, tables, ks, vs = so.paged([50, 9], 32, 2, 25)
    q = torch.randn(2, 8, 128, generator=torch.Generator().manual_seed(16)).to(BF)
    lens = torch.tensor([50, 9], dtype=torch.int32).cuda()
    got = paged_decode_attention(q.cuda(), k_cache.cuda(), v_cache.cuda(), tables.cuda(), lens,
                                 SCALE, 50)
    for i, n in enumerate((50, 9)):
        want, bound = so.attend(q[i:i + 1], ks[i], vs[i], torch.ones(1, n, dtype=torch.bool),
                                torch.zeros(1, n), scale=SCALE)
        so.check(got[i:i + 1], want, bound, "bf16 row")
    with pytest.raises(ValueError):
        paged_decode_attention(q.cuda(), k_cache.cuda(), v_cache.cuda(), tables.cuda(), lens,
                               SCALE, 50, k_scale=torch.zeros(1, device="cuda"),
                               v_scale=torch.zeros(1, device="cuda"))


def test_library_refuses_bad_device_calls():
    lib = _native.load()
    buf = np.zeros(64, dtype=np.uint8)
    assert lib.kvc_dequant_fp4(buf.ctypes.data, buf.ctypes.data, 1, 64, buf.ctypes.data, None) == -1


@pytest.mark.parametrize("decode,chunks,width", [
    ([40, 3], [(5, 700), (2, 65)], None), ([40, 3], [(5, 700), (2, 65)], 2200), ([], [(9, 90)], 2200),
    ([90, 70], [(300, 900)], None), ([33, 50], [], None)])
@pytest.mark.parametrize("native", [True, False])
def test_offsets_in_longer_tensors(decode, chunks, width, native, monkeypatch):
    """Offsets and lengths at the head of longer buffers, with table rows of others
    behind the call's: read in place whole and cut, and gathered."""
    if not native:
        monkeypatch.setattr(_native, "_host", _native._NoHostPath)
    lens = decode + [m for _, m in chunks]
    pool, tables, k, v = fo.paged(lens + [60, 80], 32, 2, seed=70 + len(lens))
    gen = torch.Generator().manual_seed(30)
    q = torch.randn(len(decode) + sum(n for n, _ in chunks), 8, 128, generator=gen).to(BF)
    cu_q, cu_k = [0], [0]
    for n, m in chunks:
        cu_q.append(cu_q[-1] + n)
        cu_k.append(cu_k[-1] + m)
    kc, vc, ks, vs = _dev(pool)
    t = torch.full((tables.size(0), width or tables.size(1)), -1, dtype=torch.int32)
    t[:, :tables.size(1)] = tables
    behind_q, behind_k = [cu_q[-1] + 1, 2], [cu_k[-1] + 60, cu_k[-1] + 140]
    got = varlen_attention(
        q.cuda(), kc, vc, scale=SCALE, block_tables=t.cuda(), num_decode_rows=len(decode),
        decode_context_lens=torch.tensor(decode + [60, 80], dtype=torch.int32).cuda(),
        cu_seqlens_q=torch.tensor(cu_q + behind_q, dtype=torch.int32).cuda(),
        cu_seqlens_k=torch.tensor(cu_k + behind_k, dtype=torch.int32).cuda(),
        cu_seqlens_q_list=cu_q, cu_seqlens_k_list=cu_k, k_scale=ks, v_scale=vs)
    want, bound = _chunk_expect(q, k, v, decode, chunks)
    fo.check(got, want, bound, f"{decode} {chunks} in longer tensors")


@pytest.mark.parametrize("native", [True, False])
def test_a_refused_step_stores_nothing(native, monkeypatch):
    """paged_decode_append_fp4 with an output, tables, lengths or a shape that the
    attention refuses: the pool is as it was."""
    if not native:
        monkeypatch.setattr(_native, "_host", _native._NoHostPath)
    pool = _empty(4, 32, 2)
    before = [t.clone() for t in pool]
    q = torch.ones(3, 8, 128, dtype=BF, device="cuda")
    key = torch.ones(3, 2, 128, dtype=BF, device="cuda")
    slots = torch.tensor([0, 40, 70], dtype=torch.int32).cuda()
    tables = torch.tensor([[0], [1], [2]], dtype=torch.int32).cuda()
    lens = torch.tensor([1, 9, 7], dtype=torch.int32).cuda()
    odd = torch.zeros(3 * 8 * 128 + 1, dtype=BF, device="cuda")[1:].view(3, 8, 128)
    base = dict(q=q, tables=tables, lens=lens, out=None)
    for bad in (dict(out=odd), dict(out=q.float()), dict(out=q[:2]), dict(tables=tables[:2]),
                dict(tables=tables.flatten()), dict(lens=lens[:2]), dict(q=q[:, :7]),
                dict(q=q.float()),
                # more keys than a table may hold, which the library alone knows
                dict(tables=tables[:, :1].expand(3, (1 << 21) + 1).contiguous())):
        a = {**base, **bad}
        with pytest.raises((ValueError, AssertionError)):
            paged_decode_append_fp4(a["q"], key, key, *pool, slots, a["tables"], a["lens"], SCALE,
                                    out=a["out"])
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(pool, before)), bad.keys()
    paged_decode_append_fp4(q, key, key, *pool, slots, tables, lens, SCALE)
    assert not torch.equal(pool[0], before[0])


def test_append_of_more_or_fewer_rows_than_are_attended(monkeypatch):
    """The appended rows need not be the attended ones: two tokens of one row, or none."""
    lens = [34, 5]
    pool, tables, k, v = fo.paged([32, 5], 32, 2, seed=80)
    wide = torch.full((2, 2), -1, dtype=torch.int32)
    wide[:, :1] = tables
    wide[0, 1] = next(b for b in range(pool[0].size(0)) if b not in tables.flatten().tolist())
    gen = torch.Generator().manual_seed(31)
    q = torch.randn(2, 8, 128, generator=gen).to(BF)
    new = torch.randn(2, 2, 128, generator=gen).to(BF)
    slots = torch.tensor([int(wide[0, 1]) * 32, int(wide[0, 1]) * 32 + 1])
    for seqs in (k, v):
        seqs[0] = torch.cat((seqs[0], fo.values(*fo.encode(new))))
    dev = _dev(pool)
    lens_t = torch.tensor(lens, dtype=torch.int32).cuda()
    want, bound = _expect(q, k, v, lens)
    got = paged_decode_append_fp4(q[:1].cuda(), new.cuda(), new.cuda(), *dev, slots.cuda(),
                                  wide[:1].cuda(), lens_t[:1], SCALE)
    fo.check(got, want[:1], bound[:1], "two tokens of one row")
    none = new[:0].cuda()
    got = paged_decode_append_fp4(q.cuda(), none, none, *dev, slots[:0].cuda(), wide.cuda(),
                                  lens_t, SCALE)
    fo.check(got, want, bound, "no new tokens")
    before = [t.clone() for t in dev]
    got = paged_decode_append_fp4(q[:0].cuda(), -new.cuda(), new.cuda(), *dev, slots.cuda(),
                                  wide[:0].cuda(), lens_t[:0], SCALE)
    assert got.shape == (0, 8, 128) and not torch.equal(dev[0], before[0])


def _far_and_near(lens, kvh, page, seed, size):
    """Keys whose scores with a query of ones differ by hundreds of binades: the first
    one near (score 0, values near 1), the others far below it, with positive values
    of `size`."""
    pool, tables, _, _ = fo.paged(lens, page, kvh, seed=seed)
    gen = torch.Generator().manual_seed(seed)
    kc, vc, ks, vs = pool
    k, v = [], []
    for i, n in enumerate(lens):
        near = torch.arange(n) == 0
        x = torch.where(near[:, None, None], 0.0, -6.0).expand(n, kvh, 128).to(BF)
        y = torch.randn(n, kvh, 128, generator=gen)
        y = torch.where(near[:, None, None], y, y.abs() * size).to(BF)
        pos = torch.arange(n)
        slot = tables[i, pos // page].long() * page + pos % page
        for codes, powers, seqs, z in ((kc, ks, k, x), (vc, vs, v, y)):
            c, p = fo.encode(z)
            codes.flatten(0, 1)[slot], powers.flatten(0, 1)[slot] = c, p
            seqs.append(fo.values(c, p))
    return pool, tables, k, v


@pytest.mark.parametrize("size", [2.0 ** 80, 2.0 ** 115])
@pytest.mark.parametrize("heads,kvh", [(3, 3), (8, 2)])
def test_weights_that_underflow_count_nothing(size, heads, kvh):
    """Keys 700 binades below the row's best one, with values of up to 2^117: what they
    add to the exact result is below 2^-500, and nothing of them may be seen in the
    kernel's, read whole and cut, by rows and by chunks.  (Counted as 2^-127 each, 699
    of them would add about 0.1; no sum of them passes 2^126.)"""
    lens = [1, 64, 90, 700]
    pool, tables, k, v = _far_and_near(lens, kvh, 32, 40 + heads, size)
    q = torch.full((4, heads, 128), 8.0).to(BF)         # scores 0 and -543
    want, bound = _expect(q, k, v, lens)
    assert float(want.abs().max()) < 8 and float(bound.max()) < 0.1
    for i, got in enumerate(_decode(pool, tables, lens, q)):
        fo.check(got, want, bound, f"{heads}/{kvh}, values of {size}, form {i}")
    chunks = [(1, 1), (2, 64), (3, 90), (5, 700)]
    q = torch.full((11, heads, 128), 8.0).to(BF)
    want, bound = _chunk_expect(q, k, v, [], chunks)
    for width in (None, 2200):
        fo.check(_chunk_call(pool, tables, [], chunks, q, "known", width), want, bound,
                 f"chunks, width {width}")
