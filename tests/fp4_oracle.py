"""The 4-bit KV encoding and attention over it, in 64 bits, and how far the kernels
may be.

encode() finds each run's power and each value's code by comparing distances over
the format's whole grid; nothing of it follows the kernels' arithmetic, and codes and
powers have to be equal.

attend() forms each row from the keys it sees alone.  Its bound per output element
counts the kernel's roundings:
  * a query element x is met as two 4-bit-mantissa parts, to 2^-21 of its row's
    largest magnitude m; products are exact and summed in fp32, twice 128 of them: a
    logit is off by scale (2^-21 m sum |k| + 256 x 2^-24 sum |q k|);
  * exp2 and its argument (fp32, arguments up to 2^7 binades from the reference):
    2^-16;
  * each weight is rounded to bf16 (half a step, 2^-8 relative), the rounded
    weights' own sum dividing them: 2^-8 sum_j w_j |v_j - out|;
  * the output is rounded to bf16: 2^-8 |out|, on top of the error before it;
  * a weight times a power of V below 2^-126 counts 0 (or, from weight 0, up to
    2^-126): 6 x 2^-126 for every key.
"""
import math

import torch

HALF_BF16 = 2.0 ** -8
GRID = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def encode(x):
    """[..., 128] -> codes uint8 [..., 64], powers uint8 [..., 4] (on the CPU)."""
    x = x.double().cpu().unflatten(-1, (4, 32))
    fine = torch.isfinite(x).all(-1)
    a = torch.where(fine[..., None], x.abs(), torch.zeros(()).double())
    top = a.amax(-1)
    power = torch.full_like(top, -126.0)
    for e in range(-126, 125):
        power = torch.where(top > 6 * 2.0 ** e, torch.full_like(top, e + 1.0), power)
    scaled = a / 2.0 ** power[..., None]
    far = (scaled[..., None] - torch.tensor(GRID, dtype=torch.float64)).abs()
    least = far.amin(-1, keepdim=True)
    near = far == least
    even = torch.tensor([True, False] * 4)
    code = torch.where((near & even).any(-1), (near & even).int().argmax(-1),
                       near.int().argmax(-1))
    code = code + 8 * (torch.signbit(x) & fine[..., None])
    code = torch.where(fine[..., None], code, torch.zeros_like(code)).flatten(-2).to(torch.uint8)
    powers = torch.where(fine, power + 127, torch.full_like(power, 255.0)).to(torch.uint8)
    return code[..., 0::2] + 16 * code[..., 1::2], powers


def values(codes, powers):
    """What codes and powers stand for, float64 [..., 128]."""
    codes, powers = codes.cpu().long(), powers.cpu().double()
    nib = torch.stack((codes % 16, codes // 16), dim=-1).flatten(-2)
    grid = torch.tensor(GRID + tuple(-g for g in GRID), dtype=torch.float64)
    power = torch.where(powers == 255, torch.full((), math.nan).double(),
                        2.0 ** (powers - 127))
    return grid[nib] * power.repeat_interleave(32, dim=-1)


def attend(q, k, v, sees, scale):
    """q [n, H, 128] bf16, k / v float64 [m, KVH, 128], sees [n, m] -> (out, bound)."""
    q, sees = q.double().cpu(), sees.cpu()
    n, heads = q.shape[:2]
    m, kvh = k.shape[:2]
    group = heads // kvh
    out = torch.zeros(n, heads, 128, dtype=torch.float64)
    bound = torch.zeros_like(out)
    if m == 0 or n == 0:
        return out, bound
    zero = torch.zeros(()).double()
    for h in range(heads):
        kh, vh = k[:, h // group], v[:, h // group]
        s = (q[:, h] @ kh.t()) * scale
        size = (q[:, h].abs() @ kh.abs().t()) * abs(scale)
        split = q[:, h].abs().amax(1, keepdim=True) * kh.abs().sum(1)[None] * abs(scale)
        s = s.masked_fill(~sees, -math.inf)
        top = s.amax(1, keepdim=True)
        w = torch.exp(s - torch.where(top == -math.inf, zero, top))
        total = w.sum(1, keepdim=True)
        w = torch.where(total == 0, zero, w / total)
        e = (256 * 2.0 ** -24 * size.masked_fill(~sees, 0).amax(1, keepdim=True)
             + 2.0 ** -21 * split.masked_fill(~sees, 0).amax(1, keepdim=True) + 2.0 ** -16)
        for a in range(0, n, 16):
            see = sees[a:a + 16, :, None]
            wv = torch.where(see, w[a:a + 16, :, None] * vh[None], zero)
            o = wv.sum(1)
            dev = torch.where(see, w[a:a + 16, :, None] * (vh[None] - o[:, None]).abs(),
                              zero).sum(1)
            out[a:a + 16, h] = o
            first = HALF_BF16 * dev + 2 * e[a:a + 16] * wv.abs().sum(1) + m * 6 * 2.0 ** -126
            bound[a:a + 16, h] = first + HALF_BF16 * (o.abs() + first)
    return out, bound


def check(got, want, bound, label):
    """Every element within its bound; not finite exactly where the oracle is not."""
    got = got.double().cpu()
    finite = torch.isfinite(want)
    assert bool((torch.isfinite(got) == finite).all()), \
        f"{label}: finite where the oracle is not, or the other way round"
    over = torch.where(finite, (got - want).abs() - bound, torch.full((), -math.inf).double())
    if over.numel():
        worst = int(over.argmax())
        print(f"[fp4] {label}: worst margin {float(over.flatten()[worst]):.3e}", flush=True)
        assert float(over.flatten()[worst]) <= 0, (
            f"{label}: element {worst} of {tuple(got.shape)}: got {float(got.flatten()[worst])}, "
            f"want {float(want.flatten()[worst])}, bound {float(bound.flatten()[worst]):.3e}")


def paged(lens, page, kvh, seed, spare=2, poison=True, scale=1.0):
    """A shuffled 4-bit pool holding `lens` tokens a sequence, everything else NaN
    runs of code 6; block tables padded with -1.  Returns (pool's four tensors,
    tables, the sequences' k and v as float64), on the CPU."""
    gen = torch.Generator().manual_seed(seed)
    need = [(n + page - 1) // page for n in lens]
    blocks = sum(need) + spare
    pool = []
    for _ in "kv":
        pool.append(torch.full((blocks, page, kvh, 64), 0x77 if poison else 0, dtype=torch.uint8))
        pool.append(torch.full((blocks, page, kvh, 4), 255 if poison else 127, dtype=torch.uint8))
    tables = torch.full((len(lens), max(need + [1])), -1, dtype=torch.int32)
    order = torch.randperm(blocks, generator=gen).to(torch.int32)
    seqs, at = ([], []), 0
    for i, n in enumerate(lens):
        tables[i, :need[i]] = order[at:at + need[i]]
        at += need[i]
        pos = torch.arange(n)
        slot = tables[i, pos // page].long() * page + pos % page if n else pos
        for side in range(2):
            x = (torch.randn(n, kvh, 128, generator=gen) * scale).to(torch.bfloat16)
            codes, powers = encode(x)
            pool[2 * side].flatten(0, 1)[slot] = codes
            pool[2 * side + 1].flatten(0, 1)[slot] = powers
            seqs[side].append(values(codes, powers))
    k, ks, v, vs = pool
    return (k, v, ks, vs), tables, seqs[0], seqs[1]


def causal(n, m):
    return torch.arange(m)[None] <= torch.arange(m - n, m)[:, None]
