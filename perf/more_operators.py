"""Performance cases of the operators around a KV cache held in 4-bit floats, and
of the step tables that the GPU builds from request lengths.

Each case is one pass through one operator:

  append  a step's keys and values quantised into the 4-bit pool
          (`kernels.kv_fp4.store_kvcache_fp4`), then read back with what was
          cached before, as a prefill reads them (`kernels.varlen.gather_kv`);
  decode  attention of one token a sequence over the 4-bit pool
          (`kernels.paged_attention.paged_decode_attention`);
  chunk   decode rows and prefill chunks over the 4-bit pool
          (`kernels.varlen.varlen_attention`);
  tables  a serving step's pages, block tables, slots, positions and offsets
          from the requests' lengths (`kernels.step_tables.build_step_tables`).

`run` computes them in plain torch operations; with `own` set it calls the
package.  Geometries are the engine's: 32 query / 4 kv heads, its two-way
tensor-parallel shard 16 / 2, and 16 / 8, head_dim 128, 256-token pages.

The 4-bit pool holds, for each token and kv head, 128 codes of one sign, two
exponent and one mantissa bit (0, 0.5, 1, 1.5, 2, 3, 4, 6 and their negatives;
two to a byte, the even dim in the low half) and one power of two for each run
of 32 dims, as a byte that is its exponent + 127 (255: the run held an infinity
or a NaN and is NaN).  The power is the smallest that takes the run's largest
magnitude to 6 or less, 2^-126 at least and 2^125 at most (finite values stay
finite); values round to the nearest code, ties to the one with an even mantissa.

A case holds plain values only.  The context lengths of a batch are spread
between `lo` and `hi` without randomness; `chunks` is a text
"queries:cached,..." with one entry per prefill sequence.
"""
import math
import os
import random
import sys

import torch

own = False

D = 128
RUN = 32                    # dims that share one power of two
PAGE = 256
SCALE = D ** -0.5
DEV = "cuda"
NO_SLOT = 2 ** 31 - 1       # of a padded token: the append skips it
LISTED_PAIRS = 34_000_000 * 32      # padded query-key pairs x query heads of the largest chunk
LISTED_KV = 524_288 * 4             # context tokens x kv heads of the largest batch
LISTED_ROWS = 16_384 * 4            # tokens x kv heads of the largest append
LISTED_TOKENS = 65_536              # tokens of the largest step's tables
GRID = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def listed():
    return [
        # The last tokens of a short chat's prompt, on the small model.
        {"name": "append-chat", "kind": "append", "kv_heads": 8, "chunks": "17:64"},
        # Four prompts' chunks behind cached prefixes.
        {"name": "append-chunks-4", "kind": "append", "kv_heads": 4,
         "chunks": "512:0,511:1536,300:4097,256:8192"},
        # A long new prompt.
        {"name": "append-prompt-16k", "kind": "append", "kv_heads": 4, "chunks": "16384:0"},
        # One user's short chat on the small model: launches and latency are all of it.
        {"name": "decode-one-chat", "kind": "decode", "heads": 16, "kv_heads": 8, "batch": 1,
         "lo": 333, "hi": 333},
        # A ragged batch.
        {"name": "decode-ragged-48", "kind": "decode", "heads": 32, "kv_heads": 4, "batch": 48,
         "lo": 1025, "hi": 8007},
        # The full batch at 4k contexts.
        {"name": "decode-64x4096", "kind": "decode", "heads": 32, "kv_heads": 4, "batch": 64,
         "lo": 4096, "hi": 4096},
        # Long contexts, which is what 4 bits are for.
        {"name": "decode-16x32768", "kind": "decode", "heads": 32, "kv_heads": 4, "batch": 16,
         "lo": 32768, "hi": 32768},
        # A short prompt's second turn on the small model.
        {"name": "chunk-chat", "kind": "chunk", "heads": 16, "kv_heads": 8, "batch": 0, "lo": 0,
         "hi": 0, "chunks": "41:333"},
        # A mixed step: a decode batch and four prompts' chunks.
        {"name": "chunk-mixed-60-4", "kind": "chunk", "heads": 32, "kv_heads": 4, "batch": 60,
         "lo": 512, "hi": 4096, "chunks": "256:0,256:768,256:1536,256:3840"},
        # One chunk of a long prompt: the largest call.
        {"name": "chunk-16k", "kind": "chunk", "heads": 32, "kv_heads": 4, "batch": 0, "lo": 0,
         "hi": 0, "chunks": "2048:14336"},
        # A decode batch's next step, one request gone.
        {"name": "tables-decode-64", "kind": "tables", "batch": 64, "lo": 512, "hi": 4096,
         "page": 256, "width": 160, "chunk": 1, "prompts": 0, "idle": 0, "finished": 1,
         "free": 64, "per_row": 1},
        # A large step: decode rows, idle ones, and the chunks of 16 prompts.
        {"name": "tables-prompts-64k", "kind": "tables", "batch": 512, "lo": 1, "hi": 30000,
         "page": 256, "width": 160, "chunk": 4096, "prompts": 16, "idle": 40, "finished": 24,
         "free": 2000, "per_row": 0},
    ]


# --- sizes ------------------------------------------------------------------

def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _draw_tables(rng):
    batch, page = _log(rng, 1, 1024), rng.choice((32, 64, 256, 256, 256))
    hi = _log(rng, 2, 30000)
    lo = max(1, int(hi * rng.choice((0.01, 0.3, 1.0))))
    per_row = rng.choice((0, 0, 0, 1, 8))
    chunk = per_row or _log(rng, 1, 8192)
    prompts = 0 if per_row else min(batch, rng.randint(0, max(1, (LISTED_TOKENS // 2) // chunk)))
    idle = rng.randint(0, batch // 4)
    most = batch * (chunk // page + 1)
    return {"kind": "tables", "batch": batch, "lo": lo, "hi": hi, "page": page,
            "width": (hi + chunk) // page + 2, "chunk": chunk, "prompts": prompts, "idle": idle,
            "finished": rng.randint(0, batch // 8), "per_row": per_row,
            # sometimes too few pages: the last requests wait
            "free": rng.choice((most, most, max(1, most // 16)))}


def draw(rng):
    """One more case: a kind, then sizes over that kind's whole range."""
    heads, kv_heads = rng.choice(((32, 4), (32, 4), (16, 2), (16, 8)))
    kind = rng.choice(("append", "append", "decode", "decode", "decode", "chunk", "chunk",
                       "tables", "tables"))
    if kind == "tables":
        return _draw_tables(rng)
    while True:
        batch, hi = _log(rng, 1, 128), _log(rng, 48, 131072)
        lo = max(1, int(hi * rng.choice((0.05, 0.25, 0.6, 1.0))))
        size = {"batch": batch, "lo": lo, "hi": hi}
        if kind == "decode":
            if batch * hi * kv_heads <= LISTED_KV:
                return {"kind": kind, "heads": heads, "kv_heads": kv_heads, **size}
            continue
        n = rng.randint(1, 6)
        chunks = [(_log(rng, 1 if kind == "append" else 17, 8192),
                   rng.choice((0, 1)) * _log(rng, 64, 16384)) for _ in range(n)]
        text = ",".join("%d:%d" % c for c in chunks)
        if kind == "append":
            if sum(q + p for q, p in chunks) * kv_heads <= LISTED_ROWS:
                return {"kind": kind, "kv_heads": kv_heads, "chunks": text}
            continue
        if rng.random() < 0.5:
            size = {"batch": 0, "lo": 0, "hi": 0}
        most_q, most_k = max(q for q, _ in chunks), max(q + p for q, p in chunks)
        if n * most_q * most_k * heads <= LISTED_PAIRS and \
                size["batch"] * size["hi"] * kv_heads <= LISTED_KV // 4:
            return {"kind": kind, "heads": heads, "kv_heads": kv_heads, **size, "chunks": text}


def _spread(lo, hi, n):
    """`n` whole numbers spread over lo .. hi (golden-ratio steps)."""
    return [lo + int(round((hi - lo) * ((i * 0.6180339887498949 + 0.5) % 1.0))) for i in range(n)]


def _chunks(case):
    return [tuple(int(x) for x in c.split(":")) for c in case["chunks"].split(",") if c]


# --- the 4-bit encoding, plain -----------------------------------------------

def _quantise(x):
    """bf16 [..., 128] -> codes uint8 [..., 64], powers uint8 [..., 4]."""
    x = x.float().unflatten(-1, (D // RUN, RUN))
    top = x.abs().amax(-1)
    fraction, power = torch.frexp(top)          # top = fraction 2^power, 1/2 <= fraction < 1
    power = torch.where(fraction > 0.75, power - 2, power - 3).clamp(-126, 125)
    fine = torch.isfinite(top)
    power = torch.where(fine & (top > 0), power, -126)
    y = torch.ldexp(x, -power[..., None])
    a = y.abs()
    code = sum((a > t if k % 2 == 0 else a >= t).to(torch.uint8)
               for k, t in enumerate((0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0)))
    code = code + torch.signbit(y).to(torch.uint8) * 8
    code = torch.where(fine[..., None], code, 0).to(torch.uint8).flatten(-2)
    return (code[..., 0::2] + code[..., 1::2] * 16,
            torch.where(fine, power + 127, 255).to(torch.uint8))


def _dequantise(codes, powers):
    """The fp32 values [..., 128] that codes and powers stand for."""
    grid = torch.tensor(GRID + tuple(-g for g in GRID), device=codes.device)
    x = torch.stack((grid[(codes & 15).int()], grid[(codes >> 4).int()]), dim=-1).flatten(-2)
    s = torch.ldexp(torch.ones((), device=codes.device), powers.int() - 127)
    s = torch.where(powers == 255, torch.nan, s)
    return (x.unflatten(-1, (D // RUN, RUN)) * s[..., None]).flatten(-2)


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


def _keys(gen, n, kv_heads):
    """Keys as they come from the rotary step: some dims run several times wider."""
    wide = torch.ones(D, device=DEV)
    wide[[5, 37, 70, 101]] = 6.0
    return (_randn(gen, n, kv_heads, D) * wide).to(torch.bfloat16)


def _pool(gen, blocks, kv_heads):
    """A filled pool, page by page as steps before have appended it."""
    rows = blocks * PAGE
    pool = {}
    for name in ("k", "v"):
        codes = torch.empty(rows, kv_heads, D // 2, dtype=torch.uint8, device=DEV)
        powers = torch.empty(rows, kv_heads, D // RUN, dtype=torch.uint8, device=DEV)
        step = 1 << 16
        for a in range(0, rows, step):
            n = min(step, rows - a)
            x = _keys(gen, n, kv_heads) if name == "k" else _randn(gen, n, kv_heads, D)
            codes[a:a + n], powers[a:a + n] = _quantise(x)
        pool[name + "_cache"] = codes.view(blocks, PAGE, kv_heads, D // 2)
        pool[name + "_scale"] = powers.view(blocks, PAGE, kv_heads, D // RUN)
    return pool


def _offsets(chunks):
    cu_q, cu_k = [0], [0]
    for c, p in chunks:
        cu_q.append(cu_q[-1] + c)
        cu_k.append(cu_k[-1] + c + p)
    return cu_q, cu_k


def _prepare_append(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    chunks, kvh = _chunks(case), case["kv_heads"]
    tables, blocks = _tables([q + p for q, p in chunks], gen)
    cu_q, cu_k = _offsets(chunks)
    n = cu_q[-1]
    row = torch.repeat_interleave(torch.arange(len(chunks), device=DEV),
                                  torch.tensor([q for q, _ in chunks], device=DEV))
    pos = torch.cat([torch.arange(p, p + q, device=DEV) for q, p in chunks])
    slots = tables[row, pos // PAGE] * PAGE + pos % PAGE
    # v is a view of the fused projection
    v = _randn(gen, n, 10 * kvh * D)[:, 9 * kvh * D:].view(n, kvh, D)
    return {"case": case, **_pool(gen, blocks, kvh), "tables": tables, "k": _keys(gen, n, kvh),
            "v": v, "slots": slots.to(torch.int32), "cu_k": _i32(cu_k), "host": {"cu_k": cu_k}}


def _prepare_rows(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    heads, kvh = case["heads"], case["kv_heads"]
    lens, chunks = _spread(case["lo"], case["hi"], case["batch"]), \
        _chunks(case) if case["kind"] == "chunk" else []
    tables, blocks = _tables(lens + [q + p for q, p in chunks], gen)
    cu_q, cu_k = _offsets(chunks)
    return {"case": case, **_pool(gen, blocks, kvh), "tables": tables,
            "q": _randn(gen, len(lens) + cu_q[-1], heads, D), "lens": _i32(lens),
            "cu_q": _i32(cu_q), "cu_k": _i32(cu_k),
            "host": {"lens": lens, "cu_q": cu_q, "cu_k": cu_k}}


def _prepare_tables(case, seed):
    rng = random.Random(seed)
    batch, page, width = case["batch"], case["page"], case["width"]
    kinds = ["finished"] * case["finished"] + ["idle"] * case["idle"] + \
        ["prompt"] * case["prompts"]
    kinds = (kinds + ["decode"] * batch)[:batch]
    rng.shuffle(kinds)
    lens = _spread(case["lo"], case["hi"], batch)
    rng.shuffle(lens)
    new = [{"finished": 0, "idle": 0, "prompt": case["chunk"],
            "decode": case["per_row"] or 1}[k] for k in kinds]
    # a row may hold a page more than it fills: drafts that were not accepted
    held = [min(width, (n + page - 1) // page + (rng.random() < 0.1)) for n in lens]
    blocks = sum((n + page - 1) // page for n in lens) + batch + case["free"]
    order = list(range(blocks))
    rng.shuffle(order)
    table, at = [], 0
    for n in held:
        table.append(order[at:at + n] + [-1] * (width - n))
        at += n
    free = (order[at:at + case["free"]] + [0] * blocks)[:blocks]
    tokens = batch * case["per_row"] if case["per_row"] else \
        case["prompts"] * case["chunk"] + batch
    return {"case": case, "lens": _i32(lens), "new": _i32(new), "held": _i32(held),
            "table": _i32(table), "free": _i32(free), "num_free": _i32([case["free"]]),
            "finished": torch.tensor([k == "finished" for k in kinds], device=DEV),
            "tokens": tokens}


def prepare(case, seed):
    return {"append": _prepare_append, "decode": _prepare_rows, "chunk": _prepare_rows,
            "tables": _prepare_tables}[case["kind"]](case, seed)


# --- one pass, plain --------------------------------------------------------

def _plain_append(st):
    slots = st["slots"].long()
    for x, name in ((st["k"], "k"), (st["v"], "v")):
        codes, powers = _quantise(x)
        st[name + "_cache"].flatten(0, 1)[slots] = codes
        st[name + "_scale"].flatten(0, 1)[slots] = powers
    t = torch.arange(st["host"]["cu_k"][-1], device=DEV)
    row = torch.searchsorted(st["cu_k"][1:], t, right=True)
    pos = t - st["cu_k"][row]
    at = st["tables"][row, pos // PAGE].long() * PAGE + pos % PAGE
    return [_dequantise(st[n + "_cache"].flatten(0, 1)[at],
                        st[n + "_scale"].flatten(0, 1)[at]).to(torch.bfloat16) for n in "kv"]


def _padded(st, first, count, most):
    """K and V, fp32 [count kv_heads, most, 128], of `count` sequences."""
    pos = torch.arange(most, device=DEV)
    at = st["tables"][first:first + count, pos // PAGE].clamp_min(0).long() * PAGE + pos % PAGE
    out = []
    for n in "kv":
        codes = st[n + "_cache"].flatten(0, 1)[at].transpose(1, 2)
        powers = st[n + "_scale"].flatten(0, 1)[at].transpose(1, 2)
        out.append(_dequantise(codes, powers).flatten(0, 1))
    return out


def _plain_attend(q, k, v, visible):
    """q fp32 [S, n, H, 128] over k, v [S KVH, m, 128]; visible [S, n, m]."""
    s, n, heads, _ = q.shape
    kvh = k.size(0) // s
    x = q.view(s, n, kvh, heads // kvh, D).permute(0, 2, 1, 3, 4).reshape(s * kvh, -1, D)
    w = torch.bmm(x, k.transpose(1, 2).contiguous()).mul_(SCALE)
    w = w.view(s, kvh, n, heads // kvh, -1)
    w.masked_fill_(~visible[:, None, :, None, :], -math.inf)
    top = w.amax(-1, keepdim=True)
    w = w.sub_(top.masked_fill(top == -math.inf, 0.0)).exp_()
    total = w.sum(-1, keepdim=True)
    o = torch.bmm(w.view(s * kvh, -1, w.size(-1)), v).view(s, kvh, n, heads // kvh, D)
    o = torch.where(total > 0, o / total, 0.0)
    return o.permute(0, 2, 1, 3, 4).reshape(s, n, heads, D)


def _plain_decode(st, rows):
    most = max(st["host"]["lens"])
    k, v = _padded(st, 0, rows, most)
    seen = torch.arange(most, device=DEV) < st["lens"][:, None]
    return _plain_attend(st["q"][:rows, None].float(), k, v, seen[:, None])[:, 0]


def _plain_rows(st):
    host, case = st["host"], st["case"]
    rows, done = len(host["lens"]), []
    if rows:
        done.append(_plain_decode(st, rows).to(torch.bfloat16))
    n = len(host["cu_q"]) - 1
    if n:
        nq = (st["cu_q"][1:] - st["cu_q"][:-1]).long()
        nk = (st["cu_k"][1:] - st["cu_k"][:-1]).long()
        most_q = max(b - a for a, b in zip(host["cu_q"], host["cu_q"][1:]))
        most_k = max(b - a for a, b in zip(host["cu_k"], host["cu_k"][1:]))
        t = torch.arange(most_q, device=DEV)
        live = t < nq[:, None]
        q = torch.zeros(n, most_q, case["heads"], D, device=DEV)
        q[live] = st["q"][rows:].float()
        k, v = _padded(st, rows, n, most_k)
        place = (nk - nq)[:, None] + t
        seen = torch.arange(most_k, device=DEV) <= place[..., None]
        done.append(_plain_attend(q, k, v, seen)[live].to(torch.bfloat16))
    return torch.cat(done)


def _plain_tables(st):
    case, table, gone = st["case"], st["table"], st["finished"]
    page, (batch, width) = case["page"], table.shape
    j = torch.arange(width, device=DEV)
    free = st["free"]
    # the pages of requests that ended go back to the top of the stack
    back = (j < st["held"][:, None]) & gone[:, None]
    to = st["num_free"].long() + back.flatten().cumsum(0) - 1
    free.scatter_(0, torch.where(back.flatten(), to, to.new_full((), free.numel() - 1)),
                  torch.where(back.flatten(), table.flatten(), free[-1]))
    top = st["num_free"] + back.sum()
    ctx, held = st["lens"].masked_fill(gone, 0), st["held"].masked_fill(gone, 0)
    pages = (ctx + st["new"] + page - 1) // page
    able = (st["new"] > 0) & (pages <= width)
    need = torch.where(able, (pages - held).clamp_min(0), 0)
    able &= (need == 0) | (need.cumsum(0) <= top)
    want = torch.where(able, st["new"], 0)
    able &= want <= case["per_row"] if case["per_row"] else want.cumsum(0) <= st["tokens"]
    got, take = torch.where(able, want, 0), torch.where(able, need, 0)
    before = take.cumsum(0) - take
    nth = j - held[:, None]
    at = (top - 1 - before[:, None] - nth).clamp(0, free.numel() - 1)
    table.copy_(torch.where((nth >= 0) & (nth < take[:, None]), free[at], table))
    seen = torch.where(got > 0, ctx + got, 0)
    zero = got.new_zeros(1)
    cu_q, cu_k = (torch.cat((zero, x.cumsum(0).int())) for x in (got, seen))
    t = torch.arange(st["tokens"], device=DEV)
    if case["per_row"]:
        row, nth = t // case["per_row"], t % case["per_row"]
    else:
        row = torch.searchsorted(cu_q[1:], t, right=True).clamp_max(batch - 1)
        nth = t - cu_q[row]
    live = nth < got[row]
    pos = torch.where(live, ctx[row] + nth, 0).long()
    slot = table[row, pos // page] * page + pos % page
    return {"slot_mapping": torch.where(live, slot, NO_SLOT).int(), "positions": pos,
            "query_lens": got.int(), "seq_lens": seen.int(), "context_lens": (ctx + got).int(),
            "cu_seqlens_q": cu_q, "cu_seqlens_k": cu_k, "num_blocks": (held + take).int(),
            "num_free": (top - take.sum()).int(), "block_tables": table, "free_blocks": free}


def _package():
    root = os.path.join(os.getcwd(), "s4000-moe-engine_amd")
    if root not in sys.path:
        sys.path.insert(0, root)
    from nanovllm_amd.kernels import kv_fp4, paged_attention, step_tables, varlen
    return kv_fp4, paged_attention, step_tables, varlen


def _own(st):
    kv_fp4, paged_attention, step_tables, varlen = _package()
    case = st["case"]
    if case["kind"] == "tables":
        s = step_tables.build_step_tables(
            st["lens"], st["new"], st["table"], st["held"], st["free"], st["num_free"],
            case["page"], st["tokens"], tokens_per_row=case["per_row"], finished=st["finished"])
        return {"slot_mapping": s.slot_mapping, "positions": s.positions,
                "query_lens": s.query_lens, "seq_lens": s.seq_lens,
                "context_lens": s.context_lens, "cu_seqlens_q": s.cu_seqlens_q,
                "cu_seqlens_k": s.cu_seqlens_k, "num_blocks": s.num_blocks,
                "num_free": s.num_free, "block_tables": st["table"], "free_blocks": st["free"]}
    if case["kind"] == "append":
        kv_fp4.store_kvcache_fp4(st["k"], st["v"], st["k_cache"], st["v_cache"], st["k_scale"],
                                 st["v_scale"], st["slots"])
        return list(varlen.gather_kv(st["k_cache"], st["v_cache"], st["tables"], st["cu_k"],
                                     st["host"]["cu_k"], k_scale=st["k_scale"],
                                     v_scale=st["v_scale"]))
    host = st["host"]
    if case["kind"] == "decode":
        return paged_attention.paged_decode_attention(
            st["q"], st["k_cache"], st["v_cache"], st["tables"], st["lens"], SCALE,
            max(host["lens"]), k_scale=st["k_scale"], v_scale=st["v_scale"])
    return varlen.varlen_attention(
        st["q"], st["k_cache"], st["v_cache"], scale=SCALE, block_tables=st["tables"],
        num_decode_rows=len(host["lens"]), decode_context_lens=st["lens"],
        cu_seqlens_q=st["cu_q"], cu_seqlens_k=st["cu_k"], cu_seqlens_q_list=host["cu_q"],
        cu_seqlens_k_list=host["cu_k"], k_scale=st["k_scale"], v_scale=st["v_scale"],
        decode_context_lens_list=host["lens"])


def run(state):
    if own:
        return _own(state)
    kind = state["case"]["kind"]
    if kind == "append":
        return _plain_append(state)
    if kind == "tables":
        return _plain_tables(state)
    return _plain_rows(state)


# --- what a pass cannot do without -------------------------------------------

def work(case):
    if case["kind"] == "tables":
        batch = case["batch"]
        tokens = batch * case["per_row"] or case["prompts"] * case["chunk"] + batch
        held = sum(_spread(case["lo"], case["hi"], batch)) // case["page"] + batch
        return {"bytes": tokens * 12 + batch * 40 + held * 4 * case["finished"] // batch,
                "flops": 0}
    row = 2 * (D // 2 + D // RUN) * case["kv_heads"]        # one token's K and V in the pool
    wide = 2 * 2 * D * case["kv_heads"]                     # and in bf16
    chunks = _chunks(case) if case["kind"] != "decode" else []
    if case["kind"] == "append":
        new, keys = sum(q for q, _ in chunks), sum(q + p for q, p in chunks)
        return {"bytes": (new + keys) * (row + wide), "flops": 0}
    lens = _spread(case["lo"], case["hi"], case["batch"])
    keys = sum(lens) + sum(q + p for q, p in chunks)
    pairs = sum(lens) + sum(q * p + q * (q + 1) // 2 for q, p in chunks)
    tokens = len(lens) + sum(q for q, _ in chunks)
    return {"bytes": keys * row + tokens * case["heads"] * 4 * D,
            "flops": 4 * D * case["heads"] * pairs}


# --- the definitions in 64 bits ----------------------------------------------

def _value(codes, powers):
    """What codes and powers stand for, from the fields of the code."""
    nibble = torch.stack((codes % 16, codes // 16), dim=-1).flatten(-2).long()
    sign, field, odd = 1.0 - 2.0 * (nibble // 8), (nibble // 2) % 4, (nibble % 2).double()
    size = torch.where(field == 0, odd * 0.5, (1 + odd * 0.5) * 2.0 ** (field.double() - 1))
    power = torch.where(powers == 255, torch.nan, 2.0 ** (powers.double() - 127))
    return sign * size * power.repeat_interleave(RUN, dim=-1)


def _nearest(x):
    """bf16 values as the 4-bit encoding holds them, by search over its grid."""
    x = x.double().unflatten(-1, (D // RUN, RUN))
    top = x.abs().amax(-1, keepdim=True)
    power = torch.full_like(top, -126.0)
    for e in range(-126, 125):
        power = torch.where(top > 6 * 2.0 ** e, e + 1.0, power)
    scaled = x.abs() / 2.0 ** power
    grid = torch.tensor(GRID, dtype=torch.float64, device=x.device)
    best, far = torch.zeros_like(scaled), scaled.clone()
    for i, g in enumerate(grid):
        away = (scaled - g).abs()
        better = away < far if i % 2 else away <= far
        best, far = torch.where(better, g, best), torch.where(better, away, far)
    return (torch.sign(x) * best * 2.0 ** power).flatten(-2)


def _cached(st, row, n):
    order = torch.arange(n, device=DEV)
    page, line = st["tables"][row].long()[order // PAGE], order % PAGE
    return [_value(st[x + "_cache"][page, line], st[x + "_scale"][page, line]) for x in "kv"]


def _exact_append(case, seed):
    st = _prepare_append(case, seed)
    keys, values, at = [], [], 0
    for i, (n, before) in enumerate(_chunks(case)):
        old_k, old_v = _cached(st, i, before)
        keys += [old_k, _nearest(st["k"][at:at + n])]
        values += [old_v, _nearest(st["v"][at:at + n])]
        at += n
    return [torch.cat(keys), torch.cat(values)]


def _exact_rows(case, seed):
    st = _prepare_rows(case, seed)
    kvh, done, at = case["kv_heads"], [], 0
    spans = [(1, m) for m in st["host"]["lens"]]
    spans += [(q, q + p) for q, p in _chunks(case)] if case["kind"] == "chunk" else []
    for i, (n, m) in enumerate(spans):
        k, v = _cached(st, i, m)
        key = torch.arange(m, device=DEV)
        out = torch.empty(n, case["heads"], D, dtype=torch.float64, device=DEV)
        for h in range(case["heads"]):
            g = h * kvh // case["heads"]
            logit = st["q"][at:at + n, h].double() @ k[:, g].t() / math.sqrt(D)
            logit = logit.masked_fill(key > key[m - n:, None], -math.inf)
            out[:, h] = torch.softmax(logit, dim=-1) @ v[:, g]
        done.append(out)
        at += n
    return torch.cat(done)


def exact(case, seed):
    if case["kind"] == "tables":
        return None                 # whole numbers only
    return (_exact_append if case["kind"] == "append" else _exact_rows)(case, seed)
