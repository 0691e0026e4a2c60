"""Rotary positions on several axes with the norm and the append
(kvc_qk_norm_mrope_store) against 64 bits.

Bound per element: the norm's factor and the rotation are fp32, a handful of
roundings of 2^-24 relative to |y1 c| + |y2 s| (sum of 128 squares 64 x 2^-24
at most, halved by the root, plus square root, division, two products, the
rotation's products and sum: under 64 x 2^-24 = 2^-18), then one rounding to
bf16: 2^-18 (|y1 c| + |y2 s|) + 2^-8 |out| (1 + 2^-18)."""
import math

import pytest
import torch

from nanovllm_amd.layers.rotary import (MultiAxisRotaryEmbedding, build_cos_sin_cache, pair_axes,
                                        qk_norm_mrope_store)

pytestmark = pytest.mark.gpu
DEV = "cuda"
EPS = 1e-6


def _oracle(x, w, positions, table, axes):
    x = x.double().cpu()
    if w is not None:
        x = x / torch.sqrt(x.square().mean(-1, keepdim=True) + EPS) * w.double().cpu()
    table = table.double().cpu()
    pos = positions.cpu().long()
    pos = torch.where(pos < 0, pos + table.size(0), pos)
    ok = (pos >= 0) & (pos < table.size(0))
    pos = torch.where(ok, pos, torch.zeros_like(pos))
    rows = table[pos]                                              # [A, N, 128]
    rows[~ok] = math.nan
    a = torch.as_tensor(axes).long().view(1, 1, 64).expand(1, pos.size(1), 64)
    c = rows[..., :64].gather(0, a)[0][:, None]
    s = rows[..., 64:].gather(0, a)[0][:, None]
    y1, y2 = x[..., :64], x[..., 64:]
    out = torch.cat((y1 * c - y2 * s, y2 * c + y1 * s), -1)
    size = torch.cat(((y1 * c).abs() + (y2 * s).abs(), (y2 * c).abs() + (y1 * s).abs()), -1)
    return out, 2.0 ** -18 * size + 2.0 ** -8 * (1 + 2.0 ** -18) * out.abs()


def _check(got, want, bound, label):
    got = got.double().cpu()
    assert bool((torch.isnan(got) == torch.isnan(want)).all()), label
    err = torch.where(torch.isnan(want), torch.zeros(()).double(), (got - want).abs())
    over = err - torch.where(torch.isnan(want), torch.zeros(()).double(), bound)
    if over.numel():
        print(f"[mrope] {label}: max error {float(err.max()):.3e}", flush=True)
        assert float(over.max()) <= 0, f"{label}: over the bound by {float(over.max()):.3e}"


def _inputs(n, heads, kvh, axes, seed, index=torch.int64, most=500):
    gen = torch.Generator().manual_seed(seed)
    qkv = torch.randn(n, (heads + 2 * kvh) * 128, generator=gen).to(torch.bfloat16).to(DEV)
    q, k, v = qkv.split((heads * 128, kvh * 128, kvh * 128), dim=-1)
    pos = torch.randint(0, most, (axes, n), generator=gen).to(index).to(DEV)
    w = [(1 + 0.1 * torch.randn(128, generator=gen)).to(torch.bfloat16).to(DEV) for _ in range(2)]
    return (q.view(n, heads, 128), k.view(n, kvh, 128), v.view(n, kvh, 128), pos, w,
            build_cos_sin_cache(128, most, 1e4, DEV))


@pytest.mark.parametrize("sections,interleaved", [((24, 20, 20), False), ((24, 20, 20), True),
                                                  ((16, 24, 24), False), ((23, 21, 20), True),
                                                  ((63, 1), True), ((1, 62, 1), False), ((64,), True),
                                                  ((16, 16, 16, 16), True), ((64, 0, 0), True)])
@pytest.mark.parametrize("heads,kvh,n", [(32, 4, 7), (16, 8, 1), (16, 2, 1026), (5, 1, 1100),
                                         (64, 8, 33), (96, 16, 1030)])
def test_norm_rotate_append(sections, interleaved, heads, kvh, n):
    q, k, v, pos, w, table = _inputs(n, heads, kvh, len(sections), n + heads)
    page, blocks = 32, (n + 31) // 32 + 2
    kc = torch.full((blocks, page, kvh, 128), 7.0, dtype=torch.bfloat16, device=DEV)
    vc = torch.full_like(kc, 9.0)
    gen = torch.Generator().manual_seed(3)
    slots = torch.randperm(blocks * page, generator=gen)[:n].to(torch.int32).to(DEV)
    qo, ko = qk_norm_mrope_store(q, k, v, pos, table, sections, interleaved, w[0], w[1], EPS,
                                 kc, vc, slots)
    torch.cuda.synchronize()
    axes = pair_axes(tuple(sections), interleaved)
    label = f"{heads}/{kvh} x {n} {sections} {interleaved}"
    _check(qo, *_oracle(q, w[0], pos, table, axes), label + " q")
    _check(ko, *_oracle(k, w[1], pos, table, axes), label + " k")
    flat_k, flat_v, at = kc.flatten(0, 1), vc.flatten(0, 1), slots.long()
    assert torch.equal(flat_k[at], ko) and torch.equal(flat_v[at], v)
    rest = torch.ones(blocks * page, dtype=torch.bool, device=DEV)
    rest[at] = False
    assert bool((flat_k[rest] == 7.0).all()) and bool((flat_v[rest] == 9.0).all())


@pytest.mark.parametrize("n", [3, 1025])
def test_positions_and_slots_out_of_range(n):
    """Negative positions and slots wrap once; past the ends a position gives
    NaN where its axis turns, a slot is skipped."""
    q, k, v, pos, w, table = _inputs(n, 8, 2, 3, 11, torch.int32, most=50)
    pos[0, 0], pos[1, 1], pos[2, 2], pos[0, n - 1] = -1, 50, -51, -50
    kc = torch.zeros(n, 1, 2, 128, dtype=torch.bfloat16, device=DEV)
    vc = torch.zeros_like(kc)
    slots = torch.arange(n, dtype=torch.int64, device=DEV)
    slots[0], slots[1] = -n, n
    qo, ko = qk_norm_mrope_store(q, k, v, pos, table, (24, 20, 20), False, w[0], w[1], EPS,
                                 kc, vc, slots)
    axes = pair_axes((24, 20, 20), False)
    _check(qo, *_oracle(q, w[0], pos, table, axes), "range q")
    _check(ko, *_oracle(k, w[1], pos, table, axes), "range k")
    want_k = ko.clone()
    want_k[1] = 0
    assert torch.equal(kc[:, 0].nan_to_num(5.0), want_k.nan_to_num(5.0))
    assert torch.equal(vc[0, 0], v[0]) and float(vc[1].abs().max()) == 0


def test_without_norm_append_or_k():
    q, k, v, pos, w, table = _inputs(19, 16, 2, 3, 12)
    qo, ko = qk_norm_mrope_store(q, k, None, pos, table, (24, 20, 20), True, return_k=False)
    assert ko is None
    axes = pair_axes((24, 20, 20), True)
    _check(qo, *_oracle(q, None, pos, table, axes), "bare")
    rope = MultiAxisRotaryEmbedding(128, 128, 500, 1e4, (24, 20, 20), True).to(DEV)
    q2, k2 = rope(pos, q.flatten(1), k.flatten(1))
    assert q2.shape == (19, 16 * 128) and torch.equal(q2.view(19, 16, 128), qo)
    _check(k2.view(19, 2, 128), *_oracle(k, None, pos, rope.cos_sin_cache, axes), "bare k")


def test_no_tokens_and_strided_positions():
    q, k, v, pos, w, table = _inputs(40, 8, 2, 3, 13)
    empty = qk_norm_mrope_store(q[:0], k[:0], None, pos[:, :0], table, (24, 20, 20))
    assert empty[0].shape == (0, 8, 128)
    cut = pos[:, 5:25]
    a, _ = qk_norm_mrope_store(q[:20], k[:20], None, cut, table, (24, 20, 20))
    b, _ = qk_norm_mrope_store(q[:20], k[:20], None, cut.contiguous(), table, (24, 20, 20))
    t, _ = qk_norm_mrope_store(q[:20], k[:20], None, cut.t().contiguous().t(), table, (24, 20, 20))
    assert torch.equal(a, b) and torch.equal(a, t)


def test_captured_and_replayed():
    q, k, v, pos, w, table = _inputs(9, 16, 2, 3, 14)
    kc = torch.zeros(4, 32, 2, 128, dtype=torch.bfloat16, device=DEV)
    vc = torch.zeros_like(kc)
    slots = torch.arange(9, dtype=torch.int32, device=DEV)

    def call(kc, vc):
        return qk_norm_mrope_store(q, k, v, pos, table, (24, 20, 20), True, w[0], w[1], EPS, kc,
                                   vc, slots, return_k=False)[0]

    call(kc, vc)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call(kc, vc)
    for step in range(3):
        q.copy_(torch.randn_like(q))
        pos.copy_(torch.randint_like(pos, 0, 500))
        slots.copy_(torch.randperm(128, device=DEV)[:9])
        graph.replay()
        k2, v2 = torch.zeros_like(kc), torch.zeros_like(vc)
        want = call(k2, v2)
        torch.cuda.synchronize()
        assert torch.equal(out, want)
        at = slots.long()
        assert torch.equal(kc.flatten(0, 1)[at], k2.flatten(0, 1)[at])
