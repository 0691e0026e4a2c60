"""Attention of drafted token trees (kvc_tree_attention) against 64 bits."""
import math
import random

import pytest
import torch

from nanovllm_amd.kernels.scored import scored_attention
from nanovllm_amd.kernels.tree import tree_attention, tree_mask_from_parents
from scored_oracle import attend, check, paged, slopes_of, tree_mask

pytestmark = pytest.mark.gpu
DEV = "cuda"
SCALE = 128 ** -0.5


def _parents(rng, n):
    return [-1 if u == 0 else rng.randrange(max(-1, u - 9), u) for u in range(n)]


def _dense(mask, n):
    u = torch.arange(n)
    return ((mask[:, u // 64] >> (u % 64)) & 1).bool()


def _queries(n, heads, seed, wide=3.0):
    gen = torch.Generator().manual_seed(seed)
    return (torch.randn(n, heads, 128, generator=gen) * wide).to(torch.bfloat16)


def _run(ctx, sizes, mask, heads, kvh, page, seed, *, cap=0.0, slopes=False, window=0,
         uniform=False, spoil=None, label=""):
    kc, vc, bt, ks, vs = paged([c + t for c, t in zip(ctx, sizes)], page, kvh, seed)
    if spoil is not None:
        spoil(kc, vc, bt, ks, vs)
    q = _queries(sum(sizes), heads, seed + 1)
    sl = slopes_of(heads) if slopes else None
    kw = {}
    if not uniform:
        cu = [0]
        for t in sizes:
            cu.append(cu[-1] + t)
        kw = dict(cu_seqlens_q=torch.tensor(cu, dtype=torch.int32, device=DEV),
                  max_seqlen_q=max(sizes))
    out = tree_attention(q.to(DEV), kc.to(DEV), vc.to(DEV), bt.to(DEV),
                         torch.tensor(ctx, dtype=torch.int32, device=DEV), mask.to(DEV), SCALE,
                         softcap=cap, alibi_slopes=sl.to(DEV) if slopes else None, window=window,
                         **kw)
    torch.cuda.synchronize()
    at, wants, bounds = 0, [], []
    for i, (c, t) in enumerate(zip(ctx, sizes)):
        sees, away = tree_mask(_dense(mask[at:at + t], t), c, window)
        w, b = attend(q[at:at + t], ks[i], vs[i], sees, away, scale=SCALE, cap=cap, slopes=sl)
        wants.append(w)
        bounds.append(b)
        at += t
    check(out, torch.cat(wants), torch.cat(bounds), label)
    return out


@pytest.mark.parametrize("form", [dict(), dict(cap=50.0), dict(slopes=True),
                                  dict(cap=30.0, slopes=True), dict(window=4),
                                  dict(window=40, slopes=True), dict(window=500, cap=20.0)])
@pytest.mark.parametrize("heads,kvh,page,most", [(32, 4, 256, 7), (16, 8, 32, 31), (16, 2, 96, 3),
                                                 (6, 2, 64, 70), (8, 1, 32, 130), (4, 4, 32, 16)])
def test_random_trees(form, heads, kvh, page, most):
    rng = random.Random(most)
    ctx = [0, 1, 31, 32, 63, 290]
    sizes = [rng.randint(1, most) for _ in ctx]
    sizes[3] = most
    mask = tree_mask_from_parents([_parents(rng, t) for t in sizes])
    _run(ctx, sizes, mask, heads, kvh, page, 40 + most, **form,
         label=f"trees {heads}/{kvh} <= {most} {form}")


def test_uniform_trees_need_no_offsets():
    rng = random.Random(1)
    sizes = [12] * 4
    mask = tree_mask_from_parents([_parents(rng, 12) for _ in sizes])
    _run([5, 0, 64, 100], sizes, mask, 16, 2, 32, 50, uniform=True, label="uniform")


def test_masks_that_are_no_trees():
    """Rows that see nothing of the tree, everything, or not themselves; bits
    past the tree's size mean nothing; a row that sees no key at all is 0."""
    sizes, ctx = [5, 3, 4], [40, 0, 33]
    mask = torch.zeros(12, 2, dtype=torch.int64)
    mask[0, 0] = 0
    mask[1, 0] = -1
    mask[2, 0] = 0b10110
    mask[3, 1] = -1
    mask[4, 0] = -(1 << 63)
    mask[6, 0] = 0b101
    mask[8, 0] = 0b1111
    mask[10, 0] = -(1 << 62)
    for form in (dict(), dict(cap=50.0), dict(slopes=True), dict(window=2)):
        out = _run(ctx, sizes, mask, 8, 2, 32, 60, **form, label=f"masks {form}")
        assert float(out[5].abs().max()) == 0.0 and float(out[7].abs().max()) == 0.0


@pytest.mark.parametrize("bad", [math.nan, math.inf])
def test_siblings_stay_out(bad):
    """Values held by branches that a token does not descend from."""
    parents = [[-1, 0, 0, 1, 1, 2, 2, 3]]
    mask = tree_mask_from_parents(parents)

    def spoil(kc, vc, bt, ks, vs):
        for u, d in ((4, 9), (6, 77)):       # leaves: their own rows alone see them
            j = 45 + u
            vs[0][j, :, d] = bad
            vc.flatten(0, 1)[int(bt[0, j // 32]) * 32 + j % 32, :, d] = bad

    out = _run([45], [8], mask, 16, 2, 32, 70, spoil=spoil, label=f"siblings {bad}")
    ok = torch.isfinite(out.float()).flatten(1).all(1).cpu().tolist()
    assert ok == [u not in (4, 6) for u in range(8)]


def test_a_chain_is_a_causal_chunk():
    """A tree without branches gives what a causal chunk gives."""
    n, ctx = 24, [100, 7]
    kc, vc, bt, ks, vs = paged([c + n for c in ctx], 32, 2, 80)
    mask = tree_mask_from_parents([list(range(-1, n - 1))] * 2)
    q = _queries(2 * n, 16, 81).to(DEV)
    args = (kc.to(DEV), vc.to(DEV))
    got = tree_attention(q, *args, bt.to(DEV), torch.tensor(ctx, dtype=torch.int32, device=DEV),
                         mask.to(DEV), SCALE, softcap=50.0)
    want = scored_attention(q, *args, scale=SCALE, block_tables=bt.to(DEV), softcap=50.0,
                            cu_seqlens_q_list=[0, n, 2 * n],
                            cu_seqlens_k_list=[0, ctx[0] + n, ctx[0] + ctx[1] + 2 * n])
    assert torch.equal(got, want)


def test_rows_past_the_offsets_are_left():
    """cu_seqlens_q on the device may cover fewer rows than q has: the rest of
    the output belongs to no sequence and is not computed from stale tables."""
    mask = tree_mask_from_parents([[-1, 0], [-1, 0, 1]])
    mask = torch.cat((mask, torch.zeros(3, 1, dtype=torch.int64)))
    kc, vc, bt, ks, vs = paged([12, 23], 32, 2, 90)
    q = _queries(8, 8, 91)
    out = tree_attention(q.to(DEV), kc.to(DEV), vc.to(DEV), bt.to(DEV),
                         torch.tensor([10, 20], dtype=torch.int32, device=DEV), mask.to(DEV),
                         SCALE, cu_seqlens_q=torch.tensor([0, 2, 5], dtype=torch.int32, device=DEV),
                         max_seqlen_q=3)
    torch.cuda.synchronize()
    at = 0
    for i, (c, t) in enumerate(((10, 2), (20, 3))):
        sees, away = tree_mask(_dense(mask[at:at + t], t), c, 0)
        check(out[at:at + t], *attend(q[at:at + t], ks[i], vs[i], sees, away, scale=SCALE), "rows")
        at += t


@pytest.mark.parametrize("form", [dict(), dict(window=3, slopes=True)])
def test_captured_step(form):
    """A captured call replayed for other contexts, masks and queries."""
    rng = random.Random(5)
    n, most = 9, [300, 300]
    kc, vc, bt, ks, vs = paged(most, 32, 2, 100, poison=False)
    kd, vd, bt_d = kc.to(DEV), vc.to(DEV), bt.to(DEV)
    q_d = torch.zeros(2 * n, 16, 128, dtype=torch.bfloat16, device=DEV)
    ctx_d = torch.zeros(2, dtype=torch.int32, device=DEV)
    mask_d = torch.zeros(2 * n, 1, dtype=torch.int64, device=DEV)
    sl = slopes_of(16) if form.get("slopes") else None
    sl_d = sl.to(DEV) if sl is not None else None

    def call():
        return tree_attention(q_d, kd, vd, bt_d, ctx_d, mask_d, SCALE, alibi_slopes=sl_d,
                              window=form.get("window", 0))

    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    for step, ctx in enumerate(([0, 291], [64, 3], [200, 200])):
        mask = tree_mask_from_parents([_parents(rng, n) for _ in ctx])
        q = _queries(2 * n, 16, 101 + step)
        q_d.copy_(q.to(DEV))
        ctx_d.copy_(torch.tensor(ctx, dtype=torch.int32))
        mask_d.copy_(mask.to(DEV))
        graph.replay()
        got = out.clone()
        eager = call()
        torch.cuda.synchronize()
        assert torch.equal(got, eager)
        for i, c in enumerate(ctx):
            sees, away = tree_mask(_dense(mask[i * n:(i + 1) * n], n), c, form.get("window", 0))
            check(got[i * n:(i + 1) * n],
                  *attend(q[i * n:(i + 1) * n], ks[i][:c + n], vs[i][:c + n], sees, away,
                          scale=SCALE, slopes=sl), f"replay {step}")


def _some_bits(size, seed):
    return random.Random(seed).getrandbits(size)


@pytest.mark.parametrize("size", [1, 3, 5, 33, 64])
@pytest.mark.parametrize("slopes", [False, True])
def test_windows_as_wide_as_the_tree(size, slopes):
    """A token that sees the whole tree is `size` places past a key whose own
    mask is empty: outside a window of `size`, inside one of `size` + 1."""
    sizes, ctx = [size] * 3, [0, 40, 31]
    mask = torch.zeros(3 * size, 1, dtype=torch.int64)
    for i in range(3):
        for t in range(1, size):
            word = (1 << size) - 1 if t == size - 1 else _some_bits(size, t + i)
            mask[i * size + t, 0] = word - (1 << 64) if word >> 63 else word
    for window in (max(1, size - 1), size, size + 1):
        out = _run(ctx, sizes, mask, 8, 2, 32, 110 + size, window=window, slopes=slopes,
                   label=f"window {window} of {size}")
        assert bool(torch.isfinite(out.float()).all())


@pytest.mark.parametrize("form", [dict(), dict(window=9), dict(slopes=True),
                                  dict(window=30, slopes=True)])
@pytest.mark.parametrize("heads,most", [(16, 7), (16, 40)])
def test_trees_past_a_short_table(form, heads, most):
    """A table that ends inside the tree, or inside its context: tokens see what
    it holds of their own paths, and nothing of another's."""
    rng = random.Random(9)
    ctx, sizes = [30, 60, 64, 100], [most] * 4
    mask = tree_mask_from_parents([_parents(rng, t) for t in sizes])
    kc, vc, bt, ks, vs = paged([c + t for c, t in zip(ctx, sizes)], 32, 2, 120)
    q = _queries(4 * most, heads, 121)
    sl = slopes_of(heads) if form.get("slopes") else None
    window = form.get("window", 0)
    out = tree_attention(q.to(DEV), kc.to(DEV), vc.to(DEV), bt[:, :2].contiguous().to(DEV),
                         torch.tensor(ctx, dtype=torch.int32, device=DEV), mask.to(DEV), SCALE,
                         alibi_slopes=None if sl is None else sl.to(DEV), window=window)
    for i, c in enumerate(ctx):
        rows = slice(i * most, (i + 1) * most)
        sees, away = tree_mask(_dense(mask[rows], most), c, window)
        w, b = attend(q[rows], ks[i][:64], vs[i][:64], sees[:, :64], away[:, :64], scale=SCALE,
                      slopes=sl)
        check(out[rows], w, b, f"short table {form} sequence {i}")
