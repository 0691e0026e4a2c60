"""Attention with shaped scores in 64 bits, and how far a bf16 kernel may be.

attend() forms each row from the keys it sees alone (values at other keys
never enter).  Its bound per output element counts the kernel's roundings:
  * each weight is rounded to bf16 (half a step, 2^-8 relative), the rounded
    weights' own sum dividing them: 2^-8 sum_j w_j |v_j - out|;
  * the output is rounded to bf16: 2^-8 |out|, on top of the error before it;
  * scores, exp2 and sums are fp32.  A logit is a sum of 128 products of bf16
    numbers, off by at most 128 x 2^-24 of their absolute sum S; shaping adds
    a few 2^-24 of the score's own size (cap, bias) and 2^-22 of the cap for
    tanh by exp2 and a reciprocal.  Every weight is then off by that relative
    error, in the numerator and in the sum: 2 e sum_j w_j |v_j|, with e from
    the row's largest S, cap and bias.
"""
import math

import torch

HALF_BF16 = 2.0 ** -8


def attend(q, k, v, sees, away, *, scale, cap=0.0, slopes=None):
    """q [n, H, 128], k / v [m, KVH, 128]; sees / away [n, m]: the mask and
    the distances |p - j|.  Returns (out, bound), float64 [n, H, 128]."""
    q, k, v = q.double().cpu(), k.double().cpu(), v.double().cpu()
    sees, away = sees.cpu(), away.double().cpu()
    n, heads = q.shape[:2]
    group = heads // k.shape[1]
    out = torch.zeros(n, heads, 128, dtype=torch.float64)
    bound = torch.zeros_like(out)
    if k.shape[0] == 0 or n == 0:
        return out, bound
    for h in range(heads):
        kh, vh = k[:, h // group], v[:, h // group]
        # keys that a row does not see may hold anything
        kz = torch.nan_to_num(kh, nan=0.0, posinf=0.0, neginf=0.0) \
            if not torch.isfinite(kh).all() else kh
        s = (q[:, h] @ kz.t()) * scale
        size = (q[:, h].abs() @ kz.abs().t()) * scale
        extra = torch.zeros(n, 1, dtype=torch.float64)
        if cap:
            s = cap * torch.tanh(s / cap)
            extra += cap * 2.0 ** -21
        if slopes is not None:
            bias = float(slopes[h]) * away
            s = s - bias
            # a key far away has no weight: count biases up to 40 (weight e^-40)
            extra += 40 * abs(float(slopes[h])) * 2.0 ** -20 + 2.0 ** -18
        s = s.masked_fill(~sees, -math.inf)
        top = s.amax(1, keepdim=True)
        w = torch.exp(s - torch.where(top == -math.inf, torch.zeros_like(top), top))
        total = w.sum(1, keepdim=True)
        w = torch.where(total > 0, w / torch.where(total > 0, total, torch.ones_like(total)),
                        torch.zeros_like(w))
        e = (128 * 2.0 ** -24 * size.masked_fill(~sees, 0).amax(1, keepdim=True) + extra
             + 2.0 ** -18)
        for a in range(0, n, 32):
            see = sees[a:a + 32, :, None]
            wv = torch.where(see, w[a:a + 32, :, None] * vh[None], torch.zeros(()).double())
            o = wv.sum(1)
            dev = torch.where(see, w[a:a + 32, :, None] * (vh[None] - o[:, None]).abs(),
                              torch.zeros(()).double()).sum(1)
            out[a:a + 32, h] = o
            first = HALF_BF16 * dev + 2 * e[a:a + 32] * wv.abs().sum(1)
            bound[a:a + 32, h] = first + HALF_BF16 * (o.abs() + first)
    return out, bound


def check(got, want, bound, label):
    """Every element within its bound; where the oracle is not finite, the
    result is not finite either."""
    got = got.double().cpu()
    finite = torch.isfinite(want)
    assert bool((torch.isfinite(got) == finite).all()), \
        f"{label}: finite where the oracle is not, or the other way round"
    err = torch.where(finite, (got - want).abs(), torch.zeros(()).double())
    over = err - torch.where(finite, bound, torch.full((), math.inf).double())
    worst = int(over.argmax()) if over.numel() else 0
    if over.numel():
        print(f"[scored] {label}: max error {float(err.max()):.3e}, "
              f"worst margin {float(over.max()):.3e}", flush=True)
        assert float(over.flatten()[worst]) <= 0, (
            f"{label}: element {worst} of {tuple(got.shape)}: got "
            f"{float(got.flatten()[worst])}, want {float(want.flatten()[worst])}, "
            f"bound {float(bound.flatten()[worst]):.3e}")


def paged(lens, page, kvh, seed, spare=2, poison=True):
    """A shuffled bf16 pool holding `lens` tokens a sequence, everything else
    NaN; block tables padded with -1.  Returns (k_cache, v_cache, tables, the
    sequences' k and v), on the CPU."""
    gen = torch.Generator().manual_seed(seed)
    need = [(n + page - 1) // page for n in lens]
    blocks = sum(need) + spare
    fill = math.nan if poison else 0.0
    k_cache = torch.full((blocks, page, kvh, 128), fill, dtype=torch.bfloat16)
    v_cache = torch.full_like(k_cache, fill)
    tables = torch.full((len(lens), max(need + [1])), -1, dtype=torch.int32)
    order = torch.randperm(blocks, generator=gen).to(torch.int32)
    ks, vs, at = [], [], 0
    for i, n in enumerate(lens):
        tables[i, :need[i]] = order[at:at + need[i]]
        at += need[i]
        k, v = (torch.randn(n, kvh, 128, generator=gen).to(torch.bfloat16) for _ in range(2))
        pos = torch.arange(n)
        slot = tables[i, pos // page].long() * page + pos % page if n else pos
        k_cache.flatten(0, 1)[slot] = k
        v_cache.flatten(0, 1)[slot] = v
        ks.append(k)
        vs.append(v)
    return k_cache, v_cache, tables, ks, vs


def slopes_of(heads):
    return torch.tensor([2.0 ** (-8.0 * (i + 1) / heads) for i in range(heads)])


def chunk_mask(n, m, window, prefix):
    p = torch.arange(m - n, m)[:, None]
    j = torch.arange(m)[None]
    sees = (j <= p) | (j < prefix)
    if window:
        sees &= p - j < window
    return sees, (p - j).abs()


def tree_mask(bits, ctx, window):
    """bits [t, t] bool (token, tree key)."""
    t = bits.shape[0]
    p = ctx + bits.sum(1) - 1
    j = torch.cat((torch.arange(ctx), p))
    sees = torch.cat((torch.ones(t, ctx, dtype=torch.bool), bits), dim=1)
    if window:
        sees &= p[:, None] - j[None] < window
    return sees, (p[:, None] - j[None]).abs()
