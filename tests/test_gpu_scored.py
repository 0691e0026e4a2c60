"""Attention with shaped scores (kvc_scored_attention) against 64 bits: caps,
distance bias, windows and two-way prefixes for decode rows, chunks and mixed
calls; odd lengths, pages and groupings; keys that a row must not see hold
NaN or infinities."""
import math

import pytest
import torch

from nanovllm_amd.kernels.scored import scored_attention
from scored_oracle import attend, check, chunk_mask, paged, slopes_of

pytestmark = pytest.mark.gpu
DEV = "cuda"
SCALE = 128 ** -0.5

FORMS = [dict(), dict(cap=50.0), dict(cap=30.0, slopes=True), dict(slopes=True), dict(cap=200.0),
         dict(window=1), dict(window=7, cap=20.0), dict(window=45), dict(window=100, slopes=True),
         dict(window=1 << 20)]
IDS = ["plain", "cap50", "cap30-distance", "distance", "cap200", "window1", "window7-cap20",
       "window45", "window100-distance", "window-all"]


def _call(q, ks, vs, k_cache, v_cache, tables, dec, chunks, *, cap=0.0, slopes=False, window=0,
          prefix=None, fresh=False, label=""):
    """dec: decode context lengths; chunks: (queries, keys) each."""
    heads = q.shape[1]
    sl = slopes_of(heads) if slopes else None
    cu_q, cu_k = [0], [0]
    for n, m in chunks:
        cu_q.append(cu_q[-1] + n)
        cu_k.append(cu_k[-1] + m)
    i32 = dict(dtype=torch.int32, device=DEV)
    kw = dict(softcap=cap, alibi_slopes=sl.to(DEV) if slopes else None, window=window)
    if prefix is not None:
        kw["prefix_lens"] = torch.tensor(prefix, **i32)
    if chunks:
        kw.update(cu_seqlens_q=torch.tensor(cu_q, **i32), cu_seqlens_k=torch.tensor(cu_k, **i32),
                  cu_seqlens_q_list=cu_q, cu_seqlens_k_list=cu_k)
    if dec:
        kw.update(num_decode_rows=len(dec), decode_context_lens=torch.tensor(dec, **i32))
    if fresh:
        out = scored_attention(q.to(DEV), None, None, scale=SCALE, k=torch.cat(ks).to(DEV),
                               v=torch.cat(vs).to(DEV), **kw)
    else:
        out = scored_attention(q.to(DEV), k_cache.to(DEV), v_cache.to(DEV), scale=SCALE,
                               block_tables=tables.to(DEV), **kw)
    torch.cuda.synchronize()
    wants, bounds, at = [], [], 0
    for i, (n, m) in enumerate([(1, c) for c in dec] + list(chunks)):
        both = prefix[i - len(dec)] if prefix is not None and i >= len(dec) else 0
        if m == 0:
            wants.append(torch.zeros(n, heads, 128).double())
            bounds.append(torch.zeros(n, heads, 128).double())
        else:
            sees, away = chunk_mask(n, m, window, both)
            w, b = attend(q[at:at + n], ks[i], vs[i], sees, away, scale=SCALE, cap=cap, slopes=sl)
            wants.append(w)
            bounds.append(b)
        at += n
    check(out, torch.cat(wants), torch.cat(bounds), label)
    return out


def _queries(n, heads, seed, wide=3.0):
    gen = torch.Generator().manual_seed(seed)
    return (torch.randn(n, heads, 128, generator=gen) * wide).to(torch.bfloat16)


@pytest.mark.parametrize("form", FORMS, ids=IDS)
@pytest.mark.parametrize("heads,kvh,page", [(32, 4, 256), (16, 8, 32), (16, 2, 96)])
def test_decode_rows(form, heads, kvh, page):
    lens = [1, 31, 0, 32, 33, 95, 96, 257, 700]
    kc, vc, bt, ks, vs = paged(lens, page, kvh, 1)
    _call(_queries(len(lens), heads, 2), ks, vs, kc, vc, bt, lens, [], **form,
          label=f"decode {heads}/{kvh} page {page} {form}")


@pytest.mark.parametrize("form", FORMS, ids=IDS)
@pytest.mark.parametrize("heads,kvh", [(8, 1), (4, 4), (6, 2)])
def test_chunks(form, heads, kvh):
    chunks = [(1, 1), (5, 5), (33, 40), (64, 300), (2, 290), (0, 64), (129, 161)]
    kc, vc, bt, ks, vs = paged([m for _, m in chunks], 64, kvh, 3)
    _call(_queries(sum(n for n, _ in chunks), heads, 4), ks, vs, kc, vc, bt, [], chunks, **form,
          label=f"chunks {heads}/{kvh} {form}")


@pytest.mark.parametrize("most", [1, 2, 4, 8, 16, 33])
@pytest.mark.parametrize("heads,kvh", [(8, 1), (16, 2), (3, 1)])
def test_every_column_width(heads, kvh, most):
    """Longest chunk x group from 3 to 264 columns: every launch form."""
    chunks = [(max(1, most - i), 200 + 37 * i) for i in range(5)]
    kc, vc, bt, ks, vs = paged([m for _, m in chunks], 32, kvh, 5)
    _call(_queries(sum(n for n, _ in chunks), heads, 6), ks, vs, kc, vc, bt, [], chunks,
          label=f"columns {heads}/{kvh} x {most}")


@pytest.mark.parametrize("form", [dict(), dict(cap=50.0), dict(slopes=True), dict(window=20),
                                  dict(window=20, slopes=True)])
@pytest.mark.parametrize("fresh", [False, True])
def test_two_way_prefix(form, fresh):
    chunks = [(70, 70), (40, 40), (33, 33), (50, 50)] if fresh else \
        [(70, 70), (40, 130), (33, 64), (50, 51)]
    prefix = [64, 40, 0, 1000]
    kc, vc, bt, ks, vs = paged([m for _, m in chunks], 32, 2, 7)
    _call(_queries(sum(n for n, _ in chunks), 8, 8), ks, vs, kc, vc, bt, [], chunks,
          prefix=prefix, fresh=fresh, **form, label=f"prefix fresh={fresh} {form}")


@pytest.mark.parametrize("form", [dict(), dict(cap=50.0, window=64)])
def test_mixed_rows(form):
    dec, chunks = [17, 300, 1], [(40, 140), (7, 7)]
    kc, vc, bt, ks, vs = paged(dec + [m for _, m in chunks], 64, 4, 9)
    _call(_queries(len(dec) + 47, 32, 10), ks, vs, kc, vc, bt, dec, chunks, prefix=[30, 7],
          **form, label=f"mixed {form}")


@pytest.mark.parametrize("cap", [0.0, 50.0])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_unseen_values_stay_out(bad, cap):
    """Keys that some rows of a tile see and others do not: the rows before
    them stay finite, whatever they hold."""
    chunks = [(40, 45), (40, 100)]
    kc, vc, bt, ks, vs = paged([45, 100], 32, 2, 11)
    for i, (n, m) in enumerate(chunks):
        for j, d in ((m - 1, 3), (m - 9, 100), (m - 20, 64)):
            vs[i][j, :, d] = bad
            vc.flatten(0, 1)[int(bt[i, j // 32]) * 32 + j % 32, :, d] = bad
        # the last key's k as well: its row alone sees it
        ks[i][m - 1, 1] = math.nan
        kc.flatten(0, 1)[int(bt[i, (m - 1) // 32]) * 32 + (m - 1) % 32, 1] = math.nan
    q = _queries(80, 8, 12)
    heads = 8
    out = scored_attention(
        q.to(DEV), kc.to(DEV), vc.to(DEV), scale=SCALE, block_tables=bt.to(DEV),
        cu_seqlens_q_list=[0, 40, 80], cu_seqlens_k_list=[0, 45, 145], softcap=cap).cpu()
    at = 0
    for i, (n, m) in enumerate(chunks):
        sees, away = chunk_mask(n, m, 0, 0)
        w, b = attend(q[at:at + n - 1], ks[i], vs[i], sees[:-1], away[:-1], scale=SCALE, cap=cap)
        check(out[at:at + n - 1], w, b, f"unseen {bad} chunk {i}")
        # the last row sees the NaN key in kv head 1
        assert not torch.isfinite(out[at + n - 1, heads // 2:]).any()
        at += n


def test_strided_rows_and_fresh_views():
    """q and v as views of a fused projection, an output of odd rows."""
    gen = torch.Generator().manual_seed(13)
    qkv = torch.randn(77, (8 + 2 * 2) * 128, generator=gen).to(torch.bfloat16).to(DEV)
    q, k, v = qkv.split((1024, 256, 256), dim=-1)
    q, k, v = q.view(77, 8, 128), k.view(77, 2, 128), v.view(77, 2, 128)
    out = scored_attention(q, None, None, scale=SCALE, k=k, v=v, softcap=30.0,
                           cu_seqlens_q_list=[0, 30, 77], cu_seqlens_k_list=[0, 30, 77])
    for a, b in ((0, 30), (30, 77)):
        sees, away = chunk_mask(b - a, b - a, 0, 0)
        check(out[a:b], *attend(q[a:b], k[a:b], v[a:b], sees, away, scale=SCALE, cap=30.0),
              "strided")


def test_bad_pages_read_as_zeros():
    """A table entry outside the pool: keys and values 0, nothing read."""
    kc, vc, bt, ks, vs = paged([100, 64], 32, 2, 14)
    bt[0, 1] = 1 << 30
    bt[1, 0] = -7
    ks[0][32:64] = 0
    vs[0][32:64] = 0
    ks[1][:32] = 0
    vs[1][:32] = 0
    _call(_queries(2, 8, 15), ks, vs, kc, vc, bt, [100, 64], [], label="bad pages")


def test_lengths_past_the_table_are_cut():
    """A context length beyond the block table reads the table's pages alone."""
    kc, vc, bt, ks, vs = paged([64, 64], 32, 2, 16)
    q = _queries(2, 8, 17)
    got = scored_attention(q.to(DEV), kc.to(DEV), vc.to(DEV), scale=SCALE, block_tables=bt.to(DEV),
                           num_decode_rows=2,
                           decode_context_lens=torch.tensor([1 << 30, 64], dtype=torch.int32,
                                                            device=DEV))
    want = scored_attention(q.to(DEV), kc.to(DEV), vc.to(DEV), scale=SCALE,
                            block_tables=bt.to(DEV), num_decode_rows=2,
                            decode_context_lens=torch.tensor([64, 64], dtype=torch.int32,
                                                             device=DEV))
    assert torch.equal(got, want)


@pytest.mark.parametrize("batch", [65, 130])
def test_many_sequences(batch):
    """More sequences than a wave has lanes, decode rows and short chunks."""
    lens = [(i * 37) % 190 + 1 for i in range(batch)]
    kc, vc, bt, ks, vs = paged(lens, 32, 1, 18)
    _call(_queries(batch, 4, 19), ks, vs, kc, vc, bt, lens, [], cap=50.0, label=f"{batch} rows")
    chunks = [(min(n, 1 + i % 5), n) for i, n in enumerate(lens)]
    _call(_queries(sum(n for n, _ in chunks), 4, 20), ks, vs, kc, vc, bt, [], chunks,
          slopes=True, label=f"{batch} chunks")


def test_long_contexts_are_split_and_joined():
    """Few rows over long contexts: every item is cut between workgroups."""
    lens = [20011, 9000]
    kc, vc, bt, ks, vs = paged(lens, 256, 1, 21)
    _call(_queries(2, 8, 22), ks, vs, kc, vc, bt, lens, [], label="long")
    _call(_queries(2, 8, 22), ks, vs, kc, vc, bt, lens, [], cap=50.0, label="long capped")
    _call(_queries(40, 2, 23), ks, vs, kc, vc, bt, [], [(33, 20011), (7, 9000)], slopes=True,
          label="long chunks")
    _call(_queries(40, 2, 23), ks, vs, kc, vc, bt, [], [(33, 20011), (7, 9000)], window=5000,
          label="long windowed chunks")


def test_offsets_past_32_bits():
    """A pool whose byte offsets pass 2^32: the last pages hold the context."""
    blocks, kvh = 4400, 4          # 4400 x 256 x 4 x 256 B = 4.6 GB each
    kc = torch.zeros(blocks, 256, kvh, 128, dtype=torch.bfloat16, device=DEV)
    vc = torch.zeros_like(kc)
    gen = torch.Generator().manual_seed(24)
    k, v = (torch.randn(300, kvh, 128, generator=gen).to(torch.bfloat16) for _ in range(2))
    bt = torch.tensor([[blocks - 1, blocks - 2]], dtype=torch.int32)
    kc[blocks - 1] = k[:256].to(DEV)
    vc[blocks - 1] = v[:256].to(DEV)
    kc[blocks - 2, :44] = k[256:].to(DEV)
    vc[blocks - 2, :44] = v[256:].to(DEV)
    q = _queries(1, 32, 25)
    out = scored_attention(q.to(DEV), kc, vc, scale=SCALE, block_tables=bt.to(DEV),
                           num_decode_rows=1, softcap=50.0,
                           decode_context_lens=torch.tensor([300], dtype=torch.int32, device=DEV))
    sees, away = chunk_mask(1, 300, 0, 0)
    check(out, *attend(q, k, v, sees, away, scale=SCALE, cap=50.0), "past 32 bits")


def test_huge_and_tiny_scores():
    """Logits of hundreds in either direction: the lazy reference holds."""
    lens = [300, 300, 300]
    kc, vc, bt, ks, vs = paged(lens, 32, 2, 26)
    for wide in (1e-3, 60.0, 400.0):
        for cap in (0.0, 50.0, 300.0):
            _call(_queries(3, 8, 27, wide), ks, vs, kc, vc, bt, lens, [], cap=cap,
                  label=f"q x {wide} cap {cap}")


def test_captured_call_replays_with_new_lengths():
    """One captured decode call serves other lengths, tables and queries, with
    eager calls of the same kernel between replays."""
    lens = [33, 400, 129]
    kc, vc, bt, ks, vs = (paged(lens, 32, 2, 28))
    kd, vd = kc.to(DEV), vc.to(DEV)
    bt_d = bt.to(DEV)
    q_d = torch.zeros(3, 8, 128, dtype=torch.bfloat16, device=DEV)
    len_d = torch.ones(3, dtype=torch.int32, device=DEV)

    def call():
        return scored_attention(q_d, kd, vd, scale=SCALE, block_tables=bt_d, num_decode_rows=3,
                                decode_context_lens=len_d, softcap=50.0)

    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    for step, now in enumerate(([33, 400, 129], [1, 1, 1], [32, 257, 64], [33, 400, 129])):
        q = _queries(3, 8, 30 + step)
        q_d.copy_(q.to(DEV))
        len_d.copy_(torch.tensor(now, dtype=torch.int32))
        graph.replay()
        got = out.clone()
        eager = call()
        torch.cuda.synchronize()
        assert torch.equal(got, eager)
        for i, m in enumerate(now):
            sees, away = chunk_mask(1, m, 0, 0)
            check(got[i:i + 1], *attend(q[i:i + 1], ks[i][:m], vs[i][:m], sees, away, scale=SCALE,
                                        cap=50.0), f"replay {step} row {i}")


def test_two_streams_at_once():
    """Calls on two streams have workspaces of their own."""
    lens = [3000, 1500]
    kc, vc, bt, ks, vs = paged(lens, 256, 1, 34)
    kd, vd, bt_d = kc.to(DEV), vc.to(DEV), bt.to(DEV)
    qs = [_queries(2, 8, 35 + i) for i in range(2)]
    len_d = torch.tensor(lens, dtype=torch.int32, device=DEV)
    q_d = [x.to(DEV) for x in qs]
    want = [scored_attention(x, kd, vd, scale=SCALE, block_tables=bt_d, num_decode_rows=2,
                             decode_context_lens=len_d) for x in q_d]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = [[], []]
    for _ in range(8):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                outs[i].append(scored_attention(q_d[i], kd, vd, scale=SCALE, block_tables=bt_d,
                                                num_decode_rows=2, decode_context_lens=len_d))
    torch.cuda.synchronize()
    for i in range(2):
        for got in outs[i]:
            assert torch.equal(got, want[i])


def test_fresh_keys_from_a_later_row():
    """cu_seqlens_k are rows of k / v and may start past the first."""
    gen = torch.Generator().manual_seed(36)
    k, v = (torch.randn(60, 2, 128, generator=gen).to(torch.bfloat16) for _ in range(2))
    q = _queries(45, 8, 37)
    out = scored_attention(q.to(DEV), None, None, scale=SCALE, k=k.to(DEV), v=v.to(DEV),
                           cu_seqlens_q_list=[0, 15, 45], cu_seqlens_k_list=[7, 25, 60])
    for a, b, c, d in ((0, 15, 7, 25), (15, 45, 25, 60)):
        w, bound = attend(q[a:b], k[c:d], v[c:d], *chunk_mask(b - a, d - c, 0, 0), scale=SCALE)
        check(out[a:b], w, bound, f"keys {c}..{d}")


@pytest.mark.parametrize("form", [dict(), dict(cap=30.0), dict(slopes=True), dict(window=40),
                                  dict(window=90, slopes=True)])
@pytest.mark.parametrize("pages", [1, 2, 4])
def test_places_past_a_short_table(form, pages):
    """Lengths beyond the block table: the keys it holds, at the places that the
    lengths give (a window may then see none of them)."""
    dec, chunks, page = [70, 128, 200], [(5, 70), (40, 129), (90, 200)], 32
    kc, vc, bt, ks, vs = paged(dec + [m for _, m in chunks], page, 2, 38)
    most = pages * page
    q = _queries(3 + 135, 8, 39)
    sl = slopes_of(8) if form.get("slopes") else None
    cap, window = form.get("cap", 0.0), form.get("window", 0)
    out = scored_attention(
        q.to(DEV), kc.to(DEV), vc.to(DEV), scale=SCALE, block_tables=bt[:, :pages].to(DEV),
        num_decode_rows=3, decode_context_lens=torch.tensor(dec, dtype=torch.int32, device=DEV),
        cu_seqlens_q_list=[0, 5, 45, 135], cu_seqlens_k_list=[0, 70, 199, 399], softcap=cap,
        alibi_slopes=None if sl is None else sl.to(DEV), window=window)
    at = 0
    for i, (n, m) in enumerate([(1, c) for c in dec] + chunks):
        sees, away = chunk_mask(n, m, window, 0)
        w, b = attend(q[at:at + n], ks[i][:most], vs[i][:most], sees[:, :most], away[:, :most],
                      scale=SCALE, cap=cap, slopes=sl)
        check(out[at:at + n], w, b, f"{pages} pages {form} sequence {i}")
        at += n
