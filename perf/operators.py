"""Performance cases of the operators for drafted trees, shaped scores and
several position axes over the paged KV cache.

Each case is one call of one operator:

  tree    attention of drafted token trees over their cached contexts
          (`kernels.tree.tree_attention`);
  score   attention whose scores are capped by a tanh or biased by distance,
          under a sliding window or a two-way prefix, for decode rows and
          prefill chunks (`kernels.scored.scored_attention`);
  mrope   q/k RMSNorm, rotary positions with three axes and the KV append
          (`layers.rotary.qk_norm_mrope_store`);
  commit  the accepted paths' rows of every layer moved to the end of their
          contexts (`kernels.tree.commit_tree_path`).

`run` computes them in plain torch operations; with `own` set it calls the
package.  Geometries are the engine's: 32 query / 4 kv heads, its two-way
tensor-parallel shard 16 / 2, and 16 / 8, head_dim 128, 256-token pages.

A case holds plain values only.  The context lengths of a batch are spread
between `lo` and `hi` without randomness, and so are its tree sizes and path
depths; `chunks` is a text "queries:cached,..." with one entry per prefill
sequence.
"""
import math
import os
import random
import sys

import torch

own = False

D = 128
HALF = D // 2
PAGE = 256
EPS = 1e-6
ROPE_BASE = 1e6
MAX_POSITION = 40960
SECTIONS = (24, 20, 20)     # rotary pairs of the time, height and width axes
SCALE = D ** -0.5
DEV = "cuda"
LISTED_PAIRS = 31_500_000 * 32      # query-key pairs x query heads of the largest chunk
LISTED_KV = 262_144 * 4             # context tokens x kv heads of the largest batch
LISTED_POOL = 64 * 3 * 28 * 4       # sequences x blocks x layers x kv heads of the largest commit
PLAIN = {"cap": 0.0, "alibi": False, "window": 0}


def listed():
    return [
        # One user's short chat on the small model, eight drafted tokens: launches
        # and latency are all of it.
        {"name": "tree-one-chat", "kind": "tree", "heads": 16, "kv_heads": 8, "batch": 1,
         "lo": 333, "hi": 333, "tokens_lo": 8, "tokens_hi": 8, **PLAIN},
        # The tensor-parallel shard of a model that caps its scores: ragged contexts,
        # ragged trees.
        {"name": "tree-tp2-capped", "kind": "tree", "heads": 16, "kv_heads": 2, "batch": 37,
         "lo": 410, "hi": 6133, "tokens_lo": 5, "tokens_hi": 31, **PLAIN, "cap": 50.0},
        # The full batch at 4k contexts, a tree of 64 tokens each.
        {"name": "tree-64x4096", "kind": "tree", "heads": 32, "kv_heads": 4, "batch": 64,
         "lo": 4096, "hi": 4096, "tokens_lo": 64, "tokens_hi": 64, **PLAIN},
        # One row of a capped model: the smallest decode call.
        {"name": "decode-one-capped", "kind": "score", "heads": 16, "kv_heads": 8, "batch": 1,
         "lo": 333, "hi": 333, "chunks": "", "prefix": 0, **PLAIN, "cap": 50.0},
        # A ragged decode batch of a model without rotary positions: a bias by distance.
        {"name": "decode-ragged-distance", "kind": "score", "heads": 32, "kv_heads": 4,
         "batch": 48, "lo": 1025, "hi": 8007, "chunks": "", "prefix": 0, **PLAIN, "alibi": True},
        # New prompts that open with an image (its patches see each other both ways).
        {"name": "prefill-image-prefix-4", "kind": "score", "heads": 32, "kv_heads": 4,
         "batch": 0, "lo": 0, "hi": 0, "chunks": "4093:0,2050:0,1300:0,749:0", "prefix": 729,
         **PLAIN},
        # Chunked prefill of a windowed, capped layer over cached prefixes.
        {"name": "prefill-window-capped-4", "kind": "score", "heads": 16, "kv_heads": 8,
         "batch": 0, "lo": 0, "hi": 0, "chunks": "512:0,511:1536,512:4097,300:8192", "prefix": 0,
         "cap": 50.0, "alibi": False, "window": 1024},
        # One chunk of a long prompt of a capped model: the largest call.
        {"name": "prefill-chunk-16k-capped", "kind": "score", "heads": 32, "kv_heads": 4,
         "batch": 0, "lo": 0, "hi": 0, "chunks": "2048:14336", "prefix": 0, **PLAIN, "cap": 50.0},
        # A decode batch's step in front of the cache, positions on three axes.
        {"name": "mrope-decode-64", "kind": "mrope", "heads": 32, "kv_heads": 4, "tokens": 64,
         "images": False, "interleaved": False},
        # A long prompt of images and text.
        {"name": "mrope-prompt-16k", "kind": "mrope", "heads": 32, "kv_heads": 4,
         "tokens": 16384, "images": True, "interleaved": True},
        # One user's accepted path, every layer of the small model.
        {"name": "commit-one", "kind": "commit", "layers": 28, "kv_heads": 8, "batch": 1,
         "lo": 333, "hi": 333, "tokens": 24, "depth_lo": 3, "depth_hi": 3},
        # A full batch's accepted paths.
        {"name": "commit-64", "kind": "commit", "layers": 28, "kv_heads": 4, "batch": 64,
         "lo": 120, "hi": 701, "tokens": 64, "depth_lo": 2, "depth_hi": 8},
    ]


# --- sizes ------------------------------------------------------------------

def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _shape(rng):
    """How a drawn model shapes its scores."""
    return {"cap": rng.choice((0.0, 0.0, 20.0, 30.0, 50.0)), "alibi": rng.random() < 0.3,
            "window": rng.choice((0, 0, 0, 1)) * _log(rng, 100, 4096)}


def draw(rng):
    """One more case: a kind, then sizes over that kind's whole range."""
    heads, kv_heads = rng.choice(((32, 4), (32, 4), (16, 2), (16, 8)))
    kind = rng.choice(("tree", "tree", "tree", "decode", "decode", "chunks", "chunks", "fresh",
                       "mixed", "mrope", "commit"))
    if kind == "mrope":
        return {"kind": "mrope", "heads": heads, "kv_heads": kv_heads,
                "tokens": _log(rng, 1, 16384), "images": rng.random() < 0.7,
                "interleaved": rng.random() < 0.5}
    if kind == "commit":
        while True:
            case = {"kind": "commit", "layers": rng.choice((28, 48)), "kv_heads": kv_heads,
                    "batch": _log(rng, 1, 64), "lo": _log(rng, 1, 700), "hi": 0,
                    "tokens": rng.randint(17, 64), "depth_lo": rng.randint(1, 4), "depth_hi": 0}
            case["hi"] = case["lo"] + rng.randint(0, 600)
            case["depth_hi"] = case["depth_lo"] + rng.randint(0, 6)
            blocks = case["batch"] * ((case["hi"] + case["tokens"]) // PAGE + 1)
            if blocks * case["layers"] * kv_heads <= LISTED_POOL:
                return case
    sizes = {"heads": heads, "kv_heads": kv_heads}
    while True:
        batch, hi = _log(rng, 1, 128), _log(rng, 48, 32768)
        lo = max(1, int(hi * rng.choice((0.05, 0.25, 0.6, 1.0))))
        size = {"batch": batch, "lo": lo, "hi": hi}
        if batch * (lo + hi) // 2 * kv_heads > LISTED_KV:
            continue
        if kind == "decode":
            return {"kind": "score", **sizes, **size, "chunks": "", "prefix": 0, **_shape(rng)}
        if kind == "tree":
            most = _log(rng, 2, 128)
            least = max(1, int(most * rng.choice((0.2, 0.6, 1.0))))
            case = {"kind": "tree", **sizes, **size, "tokens_lo": least, "tokens_hi": most,
                    **_shape(rng)}
            if batch * most <= 4096 and batch * most * (hi + most) * heads <= LISTED_PAIRS:
                return case
            continue
        n = rng.randint(1, 6)
        chunks = [(_log(rng, 17, 8192),
                   0 if kind == "fresh" else rng.choice((0, 1)) * _log(rng, 64, 16384))
                  for _ in range(n)]
        if kind == "mixed":
            batch = min(batch, 64)
            size["batch"] = batch
            if batch * (lo + hi) // 2 * kv_heads > LISTED_KV // 2:
                continue
        else:
            size = {"batch": 0, "lo": 0, "hi": 0}
        if sum(q for q, _ in chunks) > 8192 or \
                sum(q * (q + p) for q, p in chunks) * heads > LISTED_PAIRS:
            continue
        return {"kind": "score", **sizes, **size, "chunks": ",".join("%d:%d" % c for c in chunks),
                "prefix": rng.choice((0, 1)) * _log(rng, 64, 2048), **_shape(rng)}


def _spread(lo, hi, n):
    """`n` whole numbers spread over lo .. hi (golden-ratio steps)."""
    return [lo + int(round((hi - lo) * ((i * 0.6180339887498949 + 0.5) % 1.0))) for i in range(n)]


def _chunks(case):
    return [tuple(int(x) for x in c.split(":")) for c in case["chunks"].split(",") if c]


# --- inputs -----------------------------------------------------------------

def _tables(lens, gen, spare=3):
    """Block tables over a shuffled pool (-1 padded), and the pool's blocks."""
    need = [(n + PAGE - 1) // PAGE for n in lens]
    blocks = sum(need) + spare
    order = torch.randperm(blocks, generator=gen, device=DEV).to(torch.int32)
    table = torch.full((len(lens), max(need)), -1, dtype=torch.int32, device=DEV)
    at = 0
    for i, n in enumerate(need):
        table[i, :n] = order[at:at + n]
        at += n
    return table, blocks


def _randn(gen, *shape):
    return torch.randn(shape, generator=gen, device=DEV, dtype=torch.bfloat16)


def _i32(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def _slopes(case):
    """The usual geometric slopes, one per query head."""
    if not case["alibi"]:
        return None
    n = case["heads"]
    return torch.tensor([2.0 ** (-8.0 * (i + 1) / n) for i in range(n)], device=DEV)


def _queries(gen, case, n):
    """Logits about 1 wide, about 5 where a cap is there to meet them."""
    q = torch.randn(n, case["heads"], D, generator=gen, device=DEV)
    return (q * (5.0 if case["cap"] else 1.0)).to(torch.bfloat16)


def _tree(rng, n):
    """Parents (-1: the root) and, per token, the bits of its path from the root:
    a random tree whose levels widen, as a drafter's beam makes it."""
    parents, bits = [-1], [1]
    for u in range(1, n):
        parent = rng.randrange(max(0, u - 12), u)
        parents.append(parent)
        bits.append(bits[parent] | (1 << u))
    return parents, bits


def _prepare_tree(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    rng = random.Random(seed)
    lens = _spread(case["lo"], case["hi"], case["batch"])
    sizes = _spread(case["tokens_lo"], case["tokens_hi"], case["batch"])
    tables, blocks = _tables([n + t for n, t in zip(lens, sizes)], gen)
    words = (max(sizes) + 63) // 64
    mask, cu = [], [0]
    for t in sizes:
        for b in _tree(rng, t)[1]:
            row = [(b >> (64 * w)) & (2 ** 64 - 1) for w in range(words)]
            mask.append([x - 2 ** 64 if x >= 2 ** 63 else x for x in row])
        cu.append(cu[-1] + t)
    return {"case": case, "k_cache": _randn(gen, blocks, PAGE, case["kv_heads"], D),
            "v_cache": _randn(gen, blocks, PAGE, case["kv_heads"], D),
            "q": _queries(gen, case, cu[-1]), "tables": tables, "lens": _i32(lens),
            "cu_q": _i32(cu), "max_q": max(sizes),
            "mask": torch.tensor(mask, dtype=torch.int64, device=DEV), "slopes": _slopes(case),
            "host": {"lens": lens, "sizes": sizes}}


def _prepare_score(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    heads, kvh = case["heads"], case["kv_heads"]
    lens, chunks = _spread(case["lo"], case["hi"], case["batch"]), _chunks(case)
    total = lens + [q + p for q, p in chunks]
    n = len(lens) + sum(q for q, _ in chunks)
    st = {"case": case, "q": _queries(gen, case, n), "slopes": _slopes(case), "tables": None,
          "k_cache": None, "v_cache": None, "k": None, "v": None}
    fresh = not lens and all(p == 0 for _, p in chunks)
    if fresh:
        # k is the rotary step's output, v a view of the fused projection
        st["k"] = _randn(gen, n, kvh, D)
        st["v"] = _randn(gen, n, (heads + 2 * kvh) * D)[:, (heads + kvh) * D:].view(n, kvh, D)
    else:
        st["tables"], blocks = _tables(total, gen)
        st["k_cache"], st["v_cache"] = (_randn(gen, blocks, PAGE, kvh, D) for _ in range(2))
    cu_q, cu_k = [0], [0]
    for c, p in chunks:
        cu_q.append(cu_q[-1] + c)
        cu_k.append(cu_k[-1] + c + p)
    prefix = [min(c + p, case["prefix"]) for c, p in chunks] if case["prefix"] else None
    st.update(lens=_i32(lens) if lens else None, cu_q=_i32(cu_q) if chunks else None,
              cu_k=_i32(cu_k) if chunks else None, prefix=_i32(prefix) if prefix else None,
              host={"lens": lens, "cu_q": cu_q, "cu_k": cu_k, "prefix": prefix})
    return st


def _pair_axis(interleaved):
    """The axis of each rotary pair: in runs, or dealt out in turn with the
    time axis taking what is left."""
    if not interleaved:
        return [a for a, n in enumerate(SECTIONS) for _ in range(n)]
    return [i % 3 if i % 3 and i < 3 * SECTIONS[i % 3] else 0 for i in range(HALF)]


def _cos_sin():
    freq = ROPE_BASE ** -(torch.arange(HALF, dtype=torch.float64) / HALF)
    angle = torch.arange(MAX_POSITION, dtype=torch.float64)[:, None] * freq
    return torch.cat((angle.cos(), angle.sin()), dim=-1).float().to(DEV)


def _prepare_mrope(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    rng = random.Random(seed)
    heads, kvh, n = case["heads"], case["kv_heads"], case["tokens"]
    pos = torch.zeros(3, n, dtype=torch.int64)
    at, step = 0, rng.randint(0, 2000) if case["images"] else 0
    while at < n and case["images"]:
        side_h, side_w, text = rng.randint(8, 32), rng.randint(8, 32), rng.randint(20, 400)
        grid = torch.arange(side_h * side_w)
        block = torch.stack((torch.zeros_like(grid), grid // side_w, grid % side_w)) + step
        step += max(side_h, side_w)
        line = (torch.arange(text) + step).expand(3, -1)
        step += text
        block = torch.cat((block, line), dim=1)[:, :n - at]
        pos[:, at:at + block.size(1)] = block
        at += block.size(1)
    if not case["images"]:
        pos[:] = torch.tensor([rng.randint(0, MAX_POSITION - 1) for _ in range(n)])
    blocks = (n + PAGE - 1) // PAGE + 3
    q, k, v = _randn(gen, n, (heads + 2 * kvh) * D).split((heads * D, kvh * D, kvh * D), dim=-1)
    slots = torch.randperm(blocks, generator=gen, device=DEV)[torch.arange(n, device=DEV) // PAGE]
    return {"case": case, "q": q.view(n, heads, D), "k": k.view(n, kvh, D),
            "v": v.view(n, kvh, D), "positions": pos.to(DEV), "cos_sin": _cos_sin(),
            "w": (1 + 0.1 * _randn(gen, D), 1 + 0.1 * _randn(gen, D)),
            "k_cache": _randn(gen, blocks, PAGE, kvh, D), "v_cache": _randn(gen, blocks, PAGE, kvh, D),
            "slots": (slots * PAGE + torch.arange(n, device=DEV) % PAGE).to(torch.int32),
            "axis": torch.tensor(_pair_axis(case["interleaved"]), device=DEV)}


def _prepare_commit(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    rng = random.Random(seed)
    lens = _spread(case["lo"], case["hi"], case["batch"])
    depths = _spread(case["depth_lo"], case["depth_hi"], case["batch"])
    tables, blocks = _tables([n + case["tokens"] for n in lens], gen)
    most = case["depth_hi"]
    paths = []
    for d in depths:
        # the root, then one token of each level: every level is wider than the path is deep
        path = [0] + sorted(rng.sample(range(most, case["tokens"]), d - 1))
        paths.append(path + [-1] * (most - d))
    return {"case": case, "tables": tables, "lens": _i32(lens), "paths": _i32(paths),
            "depths": _i32(depths),
            "kv_cache": _randn(gen, 2, case["layers"], blocks, PAGE, case["kv_heads"], D)}


def prepare(case, seed):
    return {"tree": _prepare_tree, "score": _prepare_score, "mrope": _prepare_mrope,
            "commit": _prepare_commit}[case["kind"]](case, seed)


# --- one pass, plain --------------------------------------------------------

def _rows(pool, table_row, n):
    """The first n tokens of a sequence, through its block table, in fp32."""
    pos = torch.arange(n, device=DEV)
    return pool.flatten(0, 1)[table_row[pos // PAGE].long() * PAGE + pos % PAGE].float()


def _plain_attend(q, k, v, visible, distance, case, slopes):
    """q [n, H, D], k / v [m, KVH, D] fp32; visible(a, b) and distance(a, b)
    give the [b - a, m] masks and distances of query rows a .. b - 1."""
    n, heads = q.shape[:2]
    m, kvh = k.shape[:2]
    group = heads // kvh
    kt = k.permute(1, 2, 0).contiguous()
    vh = v.transpose(0, 1).contiguous()
    out = torch.empty(n, heads, D, device=q.device)
    step = max(1, (1 << 28) // (m * heads))
    for a in range(0, n, step):
        b = min(n, a + step)
        x = q[a:b].float().view(b - a, kvh, group, D).transpose(0, 1).reshape(kvh, -1, D)
        s = torch.bmm(x.contiguous(), kt).mul_(SCALE).view(kvh, b - a, group, m)
        if case["cap"]:
            s = s.div_(case["cap"]).tanh_().mul_(case["cap"])
        if slopes is not None:
            s -= slopes.view(kvh, 1, group, 1) * distance(a, b)[None, :, None, :].float()
        s.masked_fill_(~visible(a, b)[None, :, None, :], -math.inf)
        top = s.amax(-1, keepdim=True)
        s = s.sub_(torch.where(top == -math.inf, torch.zeros_like(top), top)).exp_()
        total = s.sum(-1, keepdim=True)
        o = torch.bmm(s.view(kvh, -1, m), vh).view(kvh, b - a, group, D)
        o = torch.where(total > 0, o / total, torch.zeros_like(o))
        out[a:b] = o.transpose(0, 1).reshape(b - a, heads, D)
    return out.to(torch.bfloat16)


def _plain_tree(st):
    case, host = st["case"], st["host"]
    out, at = torch.empty_like(st["q"]), 0
    for i, (ctx, t) in enumerate(zip(host["lens"], host["sizes"])):
        words = st["mask"][at:at + t]
        u = torch.arange(t, device=DEV)
        seen = (words[:, u // 64] >> (u % 64)) & 1
        q_pos = ctx + seen.sum(1) - 1
        k_pos = torch.cat((torch.arange(ctx, device=DEV), q_pos))
        allowed = torch.cat((torch.ones(t, ctx, dtype=torch.bool, device=DEV), seen.bool()), dim=1)
        if case["window"]:
            allowed &= q_pos[:, None] - k_pos[None, :] < case["window"]
        away = (q_pos[:, None] - k_pos[None, :]).abs()
        out[at:at + t] = _plain_attend(
            st["q"][at:at + t], _rows(st["k_cache"], st["tables"][i], ctx + t),
            _rows(st["v_cache"], st["tables"][i], ctx + t), lambda a, b: allowed[a:b],
            lambda a, b: away[a:b], case, st["slopes"])
        at += t
    return out


def _plain_score(st):
    case, host = st["case"], st["host"]
    out, at = torch.empty_like(st["q"]), 0
    n_dec = len(host["lens"])
    for i in range(n_dec + len(host["cu_q"]) - 1):
        c = i - n_dec
        n = 1 if c < 0 else host["cu_q"][c + 1] - host["cu_q"][c]
        m = host["lens"][i] if c < 0 else host["cu_k"][c + 1] - host["cu_k"][c]
        both = host["prefix"][c] if c >= 0 and host["prefix"] else 0
        if st["tables"] is None:
            k, v = (x[host["cu_k"][c]:host["cu_k"][c + 1]].float() for x in (st["k"], st["v"]))
        else:
            k, v = (_rows(x, st["tables"][i], m) for x in (st["k_cache"], st["v_cache"]))
        j = torch.arange(m, device=DEV)

        def visible(a, b):
            p = torch.arange(m - n + a, m - n + b, device=DEV)[:, None]
            ok = (j <= p) | (j < both)
            return ok & (p - j < case["window"]) if case["window"] else ok

        def distance(a, b):
            return (torch.arange(m - n + a, m - n + b, device=DEV)[:, None] - j).abs()

        out[at:at + n] = _plain_attend(st["q"][at:at + n], k, v, visible, distance, case,
                                       st["slopes"])
        at += n
    return out


def _plain_mrope(st):
    cs = st["cos_sin"][st["positions"]]                               # [3, n, D]
    axis = st["axis"].view(1, 1, HALF).expand(1, cs.size(1), HALF)
    c = cs[..., :HALF].gather(0, axis)[0][:, None]
    s = cs[..., HALF:].gather(0, axis)[0][:, None]

    def rotate(x, w):
        x = x.float()
        x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * w.float()
        a, b = x[..., :HALF], x[..., HALF:]
        return torch.cat((a * c - b * s, b * c + a * s), dim=-1).to(torch.bfloat16)

    slots = st["slots"].long()
    q = rotate(st["q"], st["w"][0])
    st["k_cache"].flatten(0, 1)[slots] = rotate(st["k"], st["w"][1])
    st["v_cache"].flatten(0, 1)[slots] = st["v"]
    return [q, st["k_cache"], st["v_cache"]]


def _plain_commit(st):
    pool = st["kv_cache"].flatten(2, 3)
    j = torch.arange(st["paths"].size(1), device=DEV)
    live = j[None] < st["depths"][:, None]

    def slots(pos):
        return st["tables"].gather(1, pos // PAGE).long() * PAGE + pos % PAGE

    src = slots((st["lens"][:, None] + st["paths"].clamp_min(0)).long())[live]
    dst = slots((st["lens"][:, None] + j[None]).long())[live]
    pool[:, :, dst] = pool[:, :, src]
    return st["kv_cache"]


def _package():
    root = os.path.join(os.getcwd(), "s4000-moe-engine_amd")
    if root not in sys.path:
        sys.path.insert(0, root)
    from nanovllm_amd.kernels import scored, tree
    from nanovllm_amd.layers import rotary
    return scored, tree, rotary


def _own(st):
    scored, tree, rotary = _package()
    case = st["case"]
    if case["kind"] == "tree":
        return tree.tree_attention(
            st["q"], st["k_cache"], st["v_cache"], st["tables"], st["lens"], st["mask"], SCALE,
            cu_seqlens_q=st["cu_q"], max_seqlen_q=st["max_q"], softcap=case["cap"],
            alibi_slopes=st["slopes"], window=case["window"])
    if case["kind"] == "score":
        host = st["host"]
        return scored.scored_attention(
            st["q"], st["k_cache"], st["v_cache"], scale=SCALE, block_tables=st["tables"],
            num_decode_rows=len(host["lens"]), decode_context_lens=st["lens"],
            cu_seqlens_q=st["cu_q"], cu_seqlens_k=st["cu_k"], cu_seqlens_q_list=host["cu_q"],
            cu_seqlens_k_list=host["cu_k"], k=st["k"], v=st["v"], softcap=case["cap"],
            alibi_slopes=st["slopes"], window=case["window"], prefix_lens=st["prefix"])
    if case["kind"] == "mrope":
        q, _ = rotary.qk_norm_mrope_store(
            st["q"], st["k"], st["v"], st["positions"], st["cos_sin"], SECTIONS,
            interleaved=case["interleaved"], q_norm_weight=st["w"][0], k_norm_weight=st["w"][1],
            eps=EPS, k_cache=st["k_cache"], v_cache=st["v_cache"], slot_mapping=st["slots"],
            return_k=False)
        return [q, st["k_cache"], st["v_cache"]]
    tree.commit_tree_path(st["kv_cache"], st["tables"], st["lens"], st["paths"], st["depths"])
    return st["kv_cache"]


def run(st):
    if own:
        return _own(st)
    return {"tree": _plain_tree, "score": _plain_score, "mrope": _plain_mrope,
            "commit": _plain_commit}[st["case"]["kind"]](st)


# --- what a pass cannot do without ------------------------------------------

def _seen(n, m, window, both):
    """Query-key pairs of n queries at the end of m keys, and the keys that any sees."""
    pairs, first = 0, m
    for p in range(m - n, m):
        low = max(0, p + 1 - window) if window else 0
        pairs += max(max(p + 1, min(both, m)) - low, 0)
        first = min(first, low)
    return pairs, m - first


def work(case):
    kvh = case["kv_heads"]
    row = 2 * kvh * D * 2                       # K and V of one token
    if case["kind"] == "mrope":
        n, heads = case["tokens"], case["heads"]
        return {"bytes": n * (2 * (heads + 2 * kvh) * D * 2 + D * 4 + 28), "flops": 0}
    lens = _spread(case["lo"], case["hi"], case["batch"])
    if case["kind"] == "commit":
        depths = _spread(case["depth_lo"], case["depth_hi"], case["batch"])
        moved = sum(depths) - len(depths)       # a path's root is where it belongs
        return {"bytes": 2 * case["layers"] * row * moved + 4 * sum(depths), "flops": 0}
    heads = case["heads"]
    if case["kind"] == "tree":
        sizes = _spread(case["tokens_lo"], case["tokens_hi"], case["batch"])
        window = case["window"]
        # every token sees its context (the window's part of it) and itself at least
        pairs = sum(t * (min(c, window - 1) if window else c) + t for c, t in zip(lens, sizes))
        keys = sum((min(c, window - 1) if window else c) + t for c, t in zip(lens, sizes))
        rows = sum(sizes)
    else:
        chunks = _chunks(case)
        parts = [_seen(1, n, case["window"], 0) for n in lens]
        parts += [_seen(c, c + p, case["window"], case["prefix"]) for c, p in chunks]
        pairs, keys = sum(p for p, _ in parts), sum(k for _, k in parts)
        rows = len(lens) + sum(c for c, _ in chunks)
    return {"bytes": keys * row + rows * 2 * heads * D * 2 + keys // PAGE * 4,
            "flops": 4 * heads * D * pairs}


# --- the same in 64 bits ----------------------------------------------------

def _exact_attend(q, k, v, q_pos, k_pos, seen, case):
    """softmax over the keys `seen` names, one query head at a time, float64."""
    n, heads = q.shape[:2]
    group = heads // k.size(1)
    out = torch.zeros(n, heads, D, dtype=torch.float64, device=DEV)
    step = max(1, (1 << 27) // k.size(0))
    for a in range(0, n, step):
        gap = q_pos[a:a + step, None] - k_pos[None]
        hide = ~seen(a, min(n, a + step))
        if case["window"]:
            hide |= gap >= case["window"]
        empty = hide.all(1)
        for h in range(heads):
            kd = k[:, h // group].double()
            logit = torch.matmul(q[a:a + step, h].double(), kd.t().contiguous()) / math.sqrt(D)
            if case["cap"]:
                logit = torch.tanh(logit / case["cap"]) * case["cap"]
            if case["alibi"]:
                logit = logit - gap.abs() * 2.0 ** (-8.0 * (h + 1) / heads)
            logit[hide] = -math.inf
            logit[empty] = 0
            weight = torch.softmax(logit, dim=1)
            weight[empty] = 0
            out[a:a + step, h] = torch.matmul(weight, v[:, h // group].double())
    return out


def _cached(st, i, n):
    order = torch.arange(n, device=DEV)
    page, line = st["tables"][i].long()[order // PAGE], order % PAGE
    return st["k_cache"][page, line], st["v_cache"][page, line]


def _exact_tree(case, seed):
    st, rng = _prepare_tree(case, seed), random.Random(seed)
    done, at = [], 0
    for i, (ctx, t) in enumerate(zip(st["host"]["lens"], st["host"]["sizes"])):
        parents, _ = _tree(rng, t)
        line = torch.zeros(t, t, dtype=torch.bool)
        depth = []
        for u, parent in enumerate(parents):
            if parent >= 0:
                line[u] = line[parent]
            line[u, u] = True
            depth.append(depth[parent] + 1 if parent >= 0 else 0)
        place = ctx + torch.tensor(depth, device=DEV)
        know = torch.ones(t, ctx + t, dtype=torch.bool, device=DEV)
        know[:, ctx:] = line.to(DEV)
        k, v = _cached(st, i, ctx + t)
        done.append(_exact_attend(st["q"][at:at + t], k, v, place,
                                  torch.cat((torch.arange(ctx, device=DEV), place)),
                                  lambda a, b: know[a:b], case))
        at += t
    return torch.cat(done)


def _exact_score(case, seed):
    st = _prepare_score(case, seed)
    host = st["host"]
    spans = [(1, m, 0) for m in host["lens"]]
    for c, (n, cached) in enumerate(_chunks(case)):
        spans.append((n, n + cached, host["prefix"][c] if host["prefix"] else 0))
    done, at, base = [], 0, 0
    for i, (n, m, both) in enumerate(spans):
        if st["tables"] is None:
            k, v = st["k"][base:base + m], st["v"][base:base + m]
            base += m
        else:
            k, v = _cached(st, i, m)
        key = torch.arange(m, device=DEV)
        pos = key[m - n:]
        done.append(_exact_attend(
            st["q"][at:at + n], k, v, pos, key,
            lambda a, b: (key[None] <= pos[a:b, None]) | (key[None] < both), case))
        at += n
    return torch.cat(done)


def _exact_mrope(case, seed):
    st = _prepare_mrope(case, seed)
    table = st["cos_sin"].double()

    def turned(x, w):
        x = x.double()
        x = x * w.double() / torch.sqrt((x * x).sum(-1, keepdim=True) / D + EPS)
        got = torch.empty_like(x)
        for i, a in enumerate(_pair_axis(case["interleaved"])):
            c, s = (table[st["positions"][a], i + off][:, None] for off in (0, HALF))
            got[..., i] = x[..., i] * c - x[..., i + HALF] * s
            got[..., i + HALF] = x[..., i + HALF] * c + x[..., i] * s
        return got

    place = st["slots"].long()
    pool_k, pool_v = st["k_cache"].double(), st["v_cache"].double()
    pool_k[place // PAGE, place % PAGE] = turned(st["k"], st["w"][1])
    pool_v[place // PAGE, place % PAGE] = st["v"].double()
    return [turned(st["q"], st["w"][0]), pool_k, pool_v]


def _exact_commit(case, seed):
    st = _prepare_commit(case, seed)
    pool, before = st["kv_cache"], {}
    moves = []
    tables, lens = st["tables"].tolist(), st["lens"].tolist()
    for i, (path, d) in enumerate(zip(st["paths"].tolist(), st["depths"].tolist())):
        for j in range(d):
            src, dst = lens[i] + path[j], lens[i] + j
            moves.append(((tables[i][src // PAGE], src % PAGE),
                          (tables[i][dst // PAGE], dst % PAGE)))
    for n, (src, _) in enumerate(moves):
        before[n] = pool[:, :, src[0], src[1]].clone()
    for n, (_, dst) in enumerate(moves):
        pool[:, :, dst[0], dst[1]] = before[n]
    return pool


def exact(case, seed):
    return {"tree": _exact_tree, "score": _exact_score, "mrope": _exact_mrope,
            "commit": _exact_commit}[case["kind"]](case, seed)
