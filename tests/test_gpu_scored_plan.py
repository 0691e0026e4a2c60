"""Shaped-score attention on both sides of every choice that the launch makes
from sizes: tables short enough to stay uncut or not, one batch entry or
several, uniform rows or offsets, more blocks than workgroups, and caps of any
size."""
import pytest
import torch

from nanovllm_amd.kernels.scored import scored_attention
from nanovllm_amd.kernels.tree import tree_attention
from scored_oracle import attend, check, chunk_mask, paged, slopes_of, tree_mask

pytestmark = pytest.mark.gpu
DEV = "cuda"
SCALE = 128 ** -0.5


def _normal(n, heads, seed, wide=2.0):
    gen = torch.Generator().manual_seed(seed)
    return (torch.randn(n, heads, 128, generator=gen) * wide).to(torch.bfloat16)


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def _chunks(q, ks, vs, chunks, label, pool=None, cap=0.0, window=0, prefix=None, most=None):
    """One call over chunks (queries, keys), from the pool or fresh."""
    cu_q, cu_k = [0], [0]
    for n, m in chunks:
        cu_q.append(cu_q[-1] + n)
        cu_k.append(cu_k[-1] + m)
    kw = dict(scale=SCALE, softcap=cap, window=window, cu_seqlens_q=_i32(cu_q),
              cu_seqlens_k=_i32(cu_k), cu_seqlens_q_list=cu_q, cu_seqlens_k_list=cu_k,
              prefix_lens=None if prefix is None else _i32(prefix))
    if pool is None:
        out = scored_attention(q.to(DEV), None, None, k=torch.cat(ks).to(DEV),
                               v=torch.cat(vs).to(DEV), **kw)
    else:
        kc, vc, bt = pool
        out = scored_attention(q.to(DEV), kc.to(DEV), vc.to(DEV), block_tables=bt.to(DEV), **kw)
    wants, bounds = [], []
    for i, (n, m) in enumerate(chunks):
        if n == 0:
            continue
        sees, away = chunk_mask(n, m, window, prefix[i] if prefix else 0)
        w, b = attend(q[cu_q[i]:cu_q[i + 1]], ks[i], vs[i], sees, away, scale=SCALE, cap=cap)
        wants.append(w)
        bounds.append(b)
    check(out, torch.cat(wants), torch.cat(bounds), label)


@pytest.mark.parametrize("pages", [1, 11, 12, 13, 23, 24, 25])
@pytest.mark.parametrize("heads,kvh", [(16, 8), (8, 1), (40, 2)])
@pytest.mark.parametrize("batch", [1, 3])
def test_decode_tables_around_the_cut(pages, heads, kvh, batch):
    lens = [32 * pages - i * 7 for i in range(batch)]
    kc, vc, bt, ks, vs = paged(lens, 32, kvh, pages)
    q = _normal(batch, heads, 1)
    out = scored_attention(q.to(DEV), kc.to(DEV), vc.to(DEV), scale=SCALE,
                           block_tables=bt.to(DEV), num_decode_rows=batch,
                           decode_context_lens=_i32(lens), softcap=50.0)
    wb = [attend(q[i:i + 1], ks[i], vs[i], *chunk_mask(1, lens[i], 0, 0), scale=SCALE, cap=50.0)
          for i in range(batch)]
    check(out, torch.cat([w for w, _ in wb]), torch.cat([b for _, b in wb]),
          f"decode of {batch}, {pages} pages, {heads}/{kvh}")


@pytest.mark.parametrize("keys", [64, 383, 385, 767, 769])
@pytest.mark.parametrize("heads,kvh", [(4, 2), (16, 2)])
def test_prompts_around_the_cut(keys, heads, kvh):
    """Fresh prompts: one, and one with an empty neighbour on either side."""
    for chunks in ([(keys, keys)], [(0, 0), (keys // 2, keys // 2), (0, 0), (1, keys - keys // 2)]):
        ks = [_normal(m, kvh, 3 + i, 1.0) for i, (_, m) in enumerate(chunks)]
        vs = [_normal(m, kvh, 9 + i, 1.0) for i, (_, m) in enumerate(chunks)]
        _chunks(_normal(sum(n for n, _ in chunks), heads, 4), ks, vs, chunks,
                f"fresh {chunks} {heads}/{kvh}")


@pytest.mark.parametrize("batch", [2, 64, 65, 130])
def test_many_short_sequences(batch):
    """As many rows as fit the card's workgroups and more, uneven chunks, an
    image prefix in some."""
    chunks = [((i * 5) % 7, 40 + (i * 13) % 57) for i in range(batch)]
    kc, vc, bt, ks, vs = paged([m for _, m in chunks], 32, 2, 5)
    prefix = [(i % 3) * 33 for i in range(batch)]
    _chunks(_normal(sum(n for n, _ in chunks), 4, 6), ks, vs, chunks, f"{batch} short chunks",
            pool=(kc, vc, bt), prefix=prefix)


@pytest.mark.parametrize("window", [1, 100, 700, 1 << 20])
def test_windows_make_long_tables_short(window):
    chunks = [(9, 2000), (17, 1400)]
    kc, vc, bt, ks, vs = paged([m for _, m in chunks], 64, 2, 7)
    _chunks(_normal(26, 8, 8), ks, vs, chunks, f"window {window}", pool=(kc, vc, bt),
            window=window, cap=30.0)


@pytest.mark.parametrize("uniform", [False, True])
@pytest.mark.parametrize("trees,tokens,ctx", [(1, 8, 300), (1, 40, 340), (3, 16, 500), (5, 64, 100),
                                              (70, 3, 60)])
def test_short_trees(uniform, trees, tokens, ctx):
    gen = torch.Generator().manual_seed(11)
    sizes = [tokens if uniform else max(1, tokens - i % 3) for i in range(trees)]
    lens = [max(0, ctx - 41 * i) for i in range(trees)]
    kc, vc, bt, ks, vs = paged([c + n for c, n in zip(lens, sizes)], 32, 2, 13)
    bits, at = [], 0
    for n in sizes:
        b = torch.eye(n, dtype=torch.bool)
        for t in range(1, n):
            b[t] |= b[int(torch.randint(0, t, (1,), generator=gen))]
        bits.append(b)
    mask = torch.zeros(sum(sizes), 1, dtype=torch.int64)
    for b in bits:
        for row in b:
            word = sum(1 << u for u in range(len(row)) if row[u])
            mask[at, 0] = word - (1 << 64) if word >> 63 else word
            at += 1
    q = _normal(sum(sizes), 8, 12)
    cu = [0]
    for n in sizes:
        cu.append(cu[-1] + n)
    kw = {} if uniform else dict(cu_seqlens_q=_i32(cu), max_seqlen_q=tokens)
    out = tree_attention(q.to(DEV), kc.to(DEV), vc.to(DEV), bt.to(DEV), _i32(lens), mask.to(DEV),
                         SCALE, **kw)
    wb = [attend(q[cu[i]:cu[i + 1]], ks[i], vs[i], *tree_mask(bits[i], lens[i], 0), scale=SCALE)
          for i in range(trees)]
    check(out, torch.cat([w for w, _ in wb]), torch.cat([b for _, b in wb]),
          f"{trees} trees of {tokens} over {ctx}")


def test_more_tokens_than_announced():
    """max_seqlen_q steers the launch only: trees longer than it, in a table
    short enough to stay uncut, are attended all the same."""
    sizes, lens = [40, 150], [100, 20]
    kc, vc, bt, ks, vs = paged([c + n for c, n in zip(lens, sizes)], 32, 2, 17)
    bits = [torch.tril(torch.ones(n, n, dtype=torch.bool)) for n in sizes]
    mask = torch.zeros(190, 3, dtype=torch.int64)
    for base, b in ((0, bits[0]), (40, bits[1])):
        for t, row in enumerate(b):
            for w in range(3):
                word = sum(1 << u for u, x in enumerate(row[64 * w:64 * w + 64].tolist()) if x)
                mask[base + t, w] = word - (1 << 64) if word >> 63 else word
    q = _normal(190, 32, 18)
    for most in (1, 8, 64):
        out = tree_attention(q.to(DEV), kc.to(DEV), vc.to(DEV), bt.to(DEV), _i32(lens),
                             mask.to(DEV), SCALE, cu_seqlens_q=_i32([0, 40, 190]),
                             max_seqlen_q=most)
        wb = [attend(q[a:b], ks[i], vs[i], *tree_mask(bits[i], lens[i], 0), scale=SCALE)
              for i, (a, b) in enumerate(((0, 40), (40, 190)))]
        check(out, torch.cat([w for w, _ in wb]), torch.cat([b for _, b in wb]),
              f"announced {most}")


@pytest.mark.parametrize("slopes", [False, True])
@pytest.mark.parametrize("cap", [1e6, 1e30])
def test_caps_far_above_the_scores(cap, slopes):
    """Such a cap changes a score by less than 2^-30 of it (z^2 / 3 with |z| <
    1e-4): the result is the uncapped one, to its bound.  Rows of one tile, of
    a few and of cut items."""
    lens = [20, 300, 2000]
    kc, vc, bt, ks, vs = paged(lens, 64, 2, 19)
    q = _normal(3, 8, 20)
    sl = slopes_of(8) if slopes else None
    out = scored_attention(q.to(DEV), kc.to(DEV), vc.to(DEV), scale=SCALE,
                           block_tables=bt.to(DEV), num_decode_rows=3,
                           decode_context_lens=_i32(lens), softcap=cap,
                           alibi_slopes=None if sl is None else sl.to(DEV))
    wb = [attend(q[i:i + 1], ks[i], vs[i], *chunk_mask(1, lens[i], 0, 0), scale=SCALE, slopes=sl)
          for i in range(3)]
    check(out, torch.cat([w for w, _ in wb]), torch.cat([b for _, b in wb]), f"cap {cap}")


@pytest.mark.parametrize("cap", [60.0, 1000.0])
def test_caps_where_series_and_exponentials_meet(cap):
    """Scores on both sides of |score| = cap / 16."""
    chunks = [(40, 70)]
    kc, vc, bt, ks, vs = paged([70], 32, 2, 21)
    for wide in (0.5, 4.0, 20.0):
        _chunks(_normal(40, 8, 22, wide), ks, vs, chunks, f"cap {cap} width {wide}",
                pool=(kc, vc, bt), cap=cap)


@pytest.mark.parametrize("form", [dict(), dict(softcap=50.0), dict(softcap=200.0),
                                  dict(alibi_slopes=True), dict(softcap=50.0, alibi_slopes=True)])
@pytest.mark.parametrize("batch,most,ctx", [(8, 8, 2500), (80, 16, 2500), (80, 31, 4000)])
def test_long_trees_of_every_width(batch, most, ctx, form):
    """64, 128 and 256 columns of one kv head, contexts long enough that items
    are cut between workgroups.  A few of the sequences against 64 bits."""
    heads = 8
    gen = torch.Generator().manual_seed(23)
    sizes = [max(1, most - i % 4) for i in range(batch)]
    lens = [ctx - (97 * i) % 400 for i in range(batch)]
    kc, vc, bt, ks, vs = paged([c + n for c, n in zip(lens, sizes)], 64, 1, 24)
    mask, bits = torch.zeros(sum(sizes), 1, dtype=torch.int64), []
    cu = [0]
    for n in sizes:
        b = torch.eye(n, dtype=torch.bool)
        for t in range(1, n):
            b[t] |= b[int(torch.randint(0, t, (1,), generator=gen))]
            mask[cu[-1] + t, 0] = sum(1 << u for u in range(n) if b[t, u])
        mask[cu[-1], 0] = 1
        bits.append(b)
        cu.append(cu[-1] + n)
    q = _normal(sum(sizes), heads, 25)
    kw = dict(form)
    sl = slopes_of(heads) if kw.pop("alibi_slopes", False) else None
    out = tree_attention(q.to(DEV), kc.to(DEV), vc.to(DEV), bt.to(DEV), _i32(lens), mask.to(DEV),
                         SCALE, cu_seqlens_q=_i32(cu), max_seqlen_q=most,
                         alibi_slopes=None if sl is None else sl.to(DEV), **kw)
    for i in range(0, batch, max(1, batch // 3)):
        sees, away = tree_mask(bits[i], lens[i], 0)
        w, b = attend(q[cu[i]:cu[i + 1]], ks[i], vs[i], sees, away, scale=SCALE,
                      cap=kw.get("softcap", 0.0), slopes=sl)
        check(out[cu[i]:cu[i + 1]], w, b, f"{batch} trees of {most} over {ctx}, sequence {i} {form}")
    assert bool(torch.isfinite(out).all())


@pytest.mark.parametrize("batch", [40, 100])
def test_uncut_items_in_several_rounds(batch):
    """Windowed chunks: several whole items a workgroup, among them sequences
    without queries.  A few of the sequences against 64 bits."""
    heads = kvh = 8
    chunks = [(0 if i % 13 == 5 else 40 - i % 9, 300 - i) for i in range(batch)]
    kc, vc, bt, ks, vs = paged([m for _, m in chunks], 32, kvh, 27)
    cu_q, cu_k = [0], [0]
    for n, m in chunks:
        cu_q.append(cu_q[-1] + n)
        cu_k.append(cu_k[-1] + m)
    q = _normal(cu_q[-1], heads, 28)
    out = scored_attention(q.to(DEV), kc.to(DEV), vc.to(DEV), scale=SCALE, window=20, softcap=50.0,
                           block_tables=bt.to(DEV), cu_seqlens_q=_i32(cu_q),
                           cu_seqlens_k=_i32(cu_k), cu_seqlens_q_list=cu_q, cu_seqlens_k_list=cu_k)
    for i in range(0, batch, 7):
        n, m = chunks[i]
        if n == 0:
            continue
        w, b = attend(q[cu_q[i]:cu_q[i + 1]], ks[i], vs[i], *chunk_mask(n, m, 20, 0), scale=SCALE,
                      cap=50.0)
        check(out[cu_q[i]:cu_q[i + 1]], w, b, f"{batch} windowed chunks, sequence {i}")
    assert bool(torch.isfinite(out).all())


def test_tables_without_pages():
    """Rows whose table holds no page at all see no key."""
    kc = torch.randn(2, 32, 2, 128).to(torch.bfloat16).to(DEV)
    tables = torch.zeros(3, 5, dtype=torch.int32, device=DEV)
    q = _normal(3, 8, 29).to(DEV)
    with pytest.raises(ValueError):
        scored_attention(q, kc, kc, scale=SCALE, block_tables=torch.zeros(
            3, 0, dtype=torch.int32, device=DEV), num_decode_rows=3,
            decode_context_lens=_i32([1, 2, 3]))
    out = scored_attention(q, kc, kc, scale=SCALE, block_tables=tables, num_decode_rows=3,
                           decode_context_lens=_i32([0, 0, 0]))
    assert not out.any()


@pytest.mark.parametrize("tokens", [1, 8, 16, 32, 64])
@pytest.mark.parametrize("cap", [20.0, 50.0, 55.0, 60.0])
@pytest.mark.parametrize("ends", ["low", "high", "rise", "fall"])
@pytest.mark.parametrize("power", [-60, 60])
def test_values_far_from_one_under_a_cap(tokens, cap, ends, power):
    """Every score at one end of the cap, or half of the keys at either: the
    weights' sums stay within fp32's range, whichever end comes first."""
    chunks = [(tokens, 300), (tokens, 1500)]
    gen = torch.Generator().manual_seed(31)
    ks, vs = [], []
    for i, (_, m) in enumerate(chunks):
        k = 1 + 0.1 * torch.randn(m, 2, 128, generator=gen)
        low = {"low": slice(0, m), "high": slice(0, 0), "rise": slice(0, m // 2),
               "fall": slice(m // 2, m)}[ends]
        k[low] *= -1
        ks.append(k.to(torch.bfloat16))
        vs.append(_normal(m, 2, 32 + i, 1.0) * 2.0 ** power)
    q = (30 * (1 + 0.1 * torch.randn(2 * tokens, 8, 128, generator=gen))).to(torch.bfloat16)
    _chunks(q, ks, vs, chunks, f"{tokens} tokens, cap {cap}, {ends}, values 2^{power}", cap=cap)
