"""The 4-bit pool under the layer, the runner and the captured step, and with the
device-built tables: the parts run together, as a serving loop uses them."""
import pytest
import torch

from nanovllm_amd.engine.graph_runner import DecodeGraphRunner
from nanovllm_amd.engine.kv_runner import KVCacheRunner
from nanovllm_amd.engine.sequence import Sequence
from nanovllm_amd.kernels.kv_fp4 import dequant_fp4, paged_decode_append_fp4
from nanovllm_amd.layers.attention import Attention
from nanovllm_amd.layers.rotary import build_cos_sin_cache
from nanovllm_amd.utils.context import get_context, reset_context, set_context
from tests import fp4_oracle as fo

pytestmark = pytest.mark.gpu
BF = torch.bfloat16
SCALE = 128 ** -0.5
HEADS, KVH, PAGE = 8, 2, 32


@pytest.fixture(autouse=True)
def _context(monkeypatch):
    monkeypatch.setattr(Sequence, "block_size", PAGE)
    yield
    reset_context()


def _runner(layers=1, blocks=24):
    runner = KVCacheRunner(layers, blocks, PAGE, KVH, 128, kv_fp4=True)
    modules = [Attention(HEADS, 128, SCALE, KVH) for _ in range(layers)]
    assert runner.bind(modules) == layers
    return runner, modules


def _rows(gen, n):
    q = torch.randn(n, HEADS, 128, generator=gen).to(BF)
    k, v = (torch.randn(n, KVH, 128, generator=gen).to(BF) for _ in range(2))
    return q, k, v


def _stored(x):
    return fo.values(*fo.encode(x))


def test_pool_of_the_runner():
    runner, (layer,) = _runner()
    assert runner.kv_cache.shape == (2, 1, 25, PAGE, KVH, 64)
    assert runner.kv_cache.dtype == torch.uint8 and runner.kv_scales.shape[-1] == 4
    assert layer.k_cache.data_ptr() == runner.kv_cache[0, 0].data_ptr()
    assert layer.v_scale.data_ptr() == runner.kv_scales[1, 0].data_ptr()
    assert not layer.kv_cache_is_int8
    bf16 = KVCacheRunner(1, 24, PAGE, KVH, 128)
    per_token = 2 * KVH * 128 * 2 / (2 * KVH * (64 + 4))
    assert bf16.kv_cache.nbytes / (runner.kv_cache.nbytes + runner.kv_scales.nbytes) == per_token


def _seq(ids, blocks, cached, new, prefill):
    s = Sequence(list(ids))
    s.block_table = list(blocks)
    s.num_cached_tokens = cached
    s.num_scheduled_tokens = new
    s.is_prefill = prefill
    return s


def test_prefill_decode_and_mixed_steps():
    """Through the runner's own producers: a prompt without a cache (attends its fresh
    keys), a chunk behind it, a decode step and a mixed step."""
    runner, (layer,) = _runner()
    gen = torch.Generator().manual_seed(1)
    hist = {}

    def run(seqs, spans, mixed=None):
        n = sum(b - a for _, a, b in spans)
        q, k, v = _rows(gen, n)
        at = 0
        for name, a, b in spans:
            old = hist.get(name, (torch.zeros(0, KVH, 128, dtype=torch.float64),) * 2)
            assert old[0].size(0) == a
            hist[name] = tuple(torch.cat((o, _stored(x[at:at + b - a])))
                               for o, x in zip(old, (k, v)))
            at += b - a
        got = layer(q.cuda().flatten(1), k.cuda().flatten(1), v.cuda().flatten(1))
        return q, k, v, got.view(n, HEADS, 128)

    a = _seq(range(40), [3, 7], 0, 40, True)
    runner.prepare_prefill([a])
    q, k, v, got = run([a], [("a", 0, 40)])
    want, bound = fo.attend(q, k.double(), v.double(), fo.causal(40, 40), SCALE)
    fo.check(got, want, bound, "fresh prompt")

    a = _seq(range(75), [3, 7, 1], 40, 35, True)
    runner.prepare_prefill([a])
    assert get_context().block_tables is not None
    q, k, v, got = run([a], [("a", 40, 75)])
    want, bound = fo.attend(q, *hist["a"], fo.causal(35, 75), SCALE)
    fo.check(got, want, bound, "chunk behind a prefix")

    a = _seq(range(76), [3, 7, 1], 75, 1, False)
    runner.prepare_decode([a])
    q, k, v, got = run([a], [("a", 75, 76)])
    want, bound = fo.attend(q, *hist["a"], fo.causal(1, 76), SCALE)
    fo.check(got, want, bound, "decode")

    a = _seq(range(77), [3, 7, 1], 76, 1, False)
    b = _seq(range(50), [5, 9], 0, 50, True)
    runner.prepare_mixed([a, b])
    q, k, v, got = run([a, b], [("a", 76, 77), ("b", 0, 50)])
    for rows, name, n, m in ((slice(0, 1), "a", 1, 77), (slice(1, 51), "b", 50, 50)):
        want, bound = fo.attend(q[rows], *hist[name], fo.causal(n, m), SCALE)
        fo.check(got[rows], want, bound, f"mixed, {name}")


def test_forward_fused_equals_its_parts():
    """The rotation runs alone and the quantising append follows, as on an int8 pool."""
    gen = torch.Generator().manual_seed(2)
    n = 5
    qkv = torch.randn(n, (HEADS + 2 * KVH) * 128, generator=gen).to(BF).cuda()
    q, k, v = qkv.split((HEADS * 128, KVH * 128, KVH * 128), dim=-1)
    cos_sin = build_cos_sin_cache(128, 64, 1e6, "cuda")
    w = [(1 + 0.1 * torch.randn(128, generator=gen)).to(BF).cuda() for _ in range(2)]
    positions = torch.tensor([3, 9, 0, 31, 40]).cuda()
    tables = torch.arange(10, dtype=torch.int32).view(5, 2).cuda()
    lens = (positions + 1).to(torch.int32)
    slots = (tables.gather(1, (positions // PAGE)[:, None]).squeeze(1) * PAGE + positions % PAGE)
    outs = []
    for fused in (True, False):
        runner, (layer,) = _runner()
        set_context(False, slot_mapping=slots.to(torch.int32), context_lens=lens,
                    block_tables=tables)
        if fused:
            out = layer.forward_fused(positions, q, k, v, cos_sin, *w, 1e-6)
        else:
            from nanovllm_amd.layers.rotary import qk_norm_rope_store
            qr, kr = qk_norm_rope_store(q.view(n, HEADS, 128), k.view(n, KVH, 128), None,
                                        positions, cos_sin, *w, 1e-6)
            out = layer(qr, kr, v.view(n, KVH, 128))
        outs.append((out, runner.kv_cache.clone(), runner.kv_scales.clone()))
    assert all(torch.equal(x, y) for x, y in zip(*outs))


def test_moves_take_codes_and_powers():
    """compact and commit_tree on a 4-bit pool."""
    runner, _ = _runner(layers=2, blocks=6)
    gen = torch.Generator(device="cuda").manual_seed(3)
    for t in (runner.kv_cache, runner.kv_scales):
        t.copy_(torch.randint(0, 255, t.shape, generator=gen, device="cuda", dtype=torch.uint8))
    before = [t.clone() for t in (runner.kv_cache, runner.kv_scales)]
    runner.compact([4, 5], [0, 1])
    for t, b in zip((runner.kv_cache, runner.kv_scales), before):
        b[:, :, [0, 1]] = b[:, :, [4, 5]]
        assert torch.equal(t, b)
    tables = torch.tensor([[2, 3]], dtype=torch.int32, device="cuda")
    runner.commit_tree(tables, torch.tensor([30], dtype=torch.int32, device="cuda"),
                       torch.tensor([[0, 2, 5]], dtype=torch.int32, device="cuda"),
                       torch.tensor([3], dtype=torch.int32, device="cuda"))
    for t, b in zip((runner.kv_cache, runner.kv_scales), before):
        rows = b[:, :, [2, 3]].flatten(2, 3)
        rows[:, :, 30:33] = rows[:, :, [30, 32, 35]]
        b[:, :, [2, 3]] = rows.view(b[:, :, [2, 3]].shape)
        assert torch.equal(t, b)


@pytest.mark.parametrize("layers,max_bs", [(1, 5), (2, 3)])
def test_captured_decode_step(layers, max_bs):
    """DecodeGraphRunner over a 4-bit pool equals the eager calls, outputs and pool
    bytes, over steps of different batches."""
    runner, _ = _runner(layers=layers, blocks=20)
    runner.kv_scales[:, :, :20] = 255            # nothing unwritten may be read
    eager = KVCacheRunner(layers, 20, PAGE, KVH, 128, kv_fp4=True)
    eager.kv_cache.copy_(runner.kv_cache), eager.kv_scales.copy_(runner.kv_scales)
    graphs = DecodeGraphRunner.from_kv_runner(runner, HEADS, max_bs, 3, SCALE, [max_bs - 2, max_bs])
    graphs.capture()
    gen = torch.Generator().manual_seed(4)
    tables = torch.randperm(18, generator=gen)[:max_bs * 3].view(max_bs, 3).to(torch.int32).cuda()
    lens = [0] * max_bs
    for step in range(40):
        bs = max_bs - step % 2 * (max_bs > 1)
        pos = lens[:bs]
        for b in range(bs):
            lens[b] += 1
        q = torch.randn(layers, bs, HEADS, 128, generator=gen).to(BF).cuda()
        k, v = (torch.randn(layers, bs, KVH, 128, generator=gen).to(BF).cuda() for _ in range(2))
        slots = torch.tensor([int(tables[b, p // PAGE]) * PAGE + p % PAGE
                              for b, p in enumerate(pos)], dtype=torch.int32).cuda()
        cl = torch.tensor(lens[:bs], dtype=torch.int32).cuda()
        got = graphs.run(q, k, v, slots, cl, tables[:bs])
        for i in range(layers):
            want = paged_decode_append_fp4(
                q[i], k[i], v[i], eager.kv_cache[0, i], eager.kv_cache[1, i],
                eager.kv_scales[0, i], eager.kv_scales[1, i], slots, tables[:bs], cl, SCALE)
            assert torch.equal(got[i], want), (step, i)
    torch.cuda.synchronize()
    assert torch.equal(runner.kv_cache[:, :, :20], eager.kv_cache[:, :, :20])
    assert torch.equal(runner.kv_scales[:, :, :20], eager.kv_scales[:, :, :20])


@pytest.mark.parametrize("capture", [False, True])
def test_serving_loop_without_the_host(capture):
    """Tables, append and attention of a decode loop whose lengths live on the device,
    eager and as one graph that is replayed; a request ends, another takes its row, and
    with the pool full a row waits."""
    rows = 3
    runner, (layer,) = _runner(blocks=4)
    tables = runner.device_tables(rows, 3)
    gen = torch.Generator().manual_seed(5)
    q = torch.zeros(rows, HEADS, 128, dtype=BF, device="cuda")
    k, v = (torch.zeros(rows, KVH, 128, dtype=BF, device="cuda") for _ in range(2))
    new = torch.ones(rows, dtype=torch.int32, device="cuda")
    finished = torch.zeros(rows, dtype=torch.bool, device="cuda")
    out = tables.outputs(rows)
    result = torch.zeros_like(q)

    def step():
        runner.prepare_decode_device(tables, new, finished, out)
        result.copy_(layer(q, k, v).view(rows, HEADS, 128))

    graph = None
    if capture:
        state = [tables.context_lens, tables.num_blocks, tables.block_tables, tables.free_blocks,
                 tables.num_free]
        saved = [x.clone() for x in state]
        step()
        torch.cuda.synchronize()
        for x, s in zip(state, saved):
            x.copy_(s)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            step()
    none = torch.zeros(0, KVH, 128, dtype=torch.float64)
    hist = [(none, none)] * rows
    waited = 0
    for i in range(75):
        gone = [i == 50 and b == 1 for b in range(rows)]
        finished.copy_(torch.tensor(gone))
        nq, nk, nv = _rows(gen, rows)
        q.copy_(nq), k.copy_(nk), v.copy_(nv)
        if graph is not None:
            graph.replay()
        else:
            step()
        torch.cuda.synchronize()
        granted = out.query_lens.tolist()
        for b in range(rows):
            if gone[b]:
                hist[b] = (none, none)
            if granted[b]:
                hist[b] = (torch.cat((hist[b][0], _stored(nk[b:b + 1]))),
                           torch.cat((hist[b][1], _stored(nv[b:b + 1]))))
            else:
                waited += 1
                assert not result[b].any()
            assert int(tables.context_lens[b]) == len(hist[b][0])
            if granted[b] and i % 6 == 0:
                want, bound = fo.attend(nq[b:b + 1], *hist[b], fo.causal(1, len(hist[b][0])),
                                        SCALE)
                fo.check(result[b:b + 1], want, bound, f"step {i}, row {b}")
    assert waited > 0                              # 4 pages for three rows of 2 and more
    # what the pool holds of row 0 is what was appended
    n = len(hist[0][0])
    pos = torch.arange(n)
    slot = (tables.block_tables[0].cpu()[pos // PAGE].long() * PAGE + pos % PAGE).cuda()
    got = dequant_fp4(layer.k_cache.flatten(0, 1)[slot], layer.k_scale.flatten(0, 1)[slot])
    assert torch.equal(got.cpu(), hist[0][0].to(BF))


@pytest.mark.parametrize("kvh,capture", [(2, False), (4, False), (4, True)])
def test_serving_loop_over_a_bf16_pool(kvh, capture):
    """The same loop over a bf16 pool, where the append may ride in the decode launch:
    rows that wait give NaN and leave the pool as it was."""
    rows, heads = 3, 2 * kvh
    runner = KVCacheRunner(1, 4, PAGE, kvh, 128)
    runner.kv_cache.zero_()
    layer = Attention(heads, 128, SCALE, kvh)
    assert runner.bind([layer]) == 1
    tables = runner.device_tables(rows, 3)
    gen = torch.Generator().manual_seed(6)
    q = torch.zeros(rows, heads, 128, dtype=BF, device="cuda")
    k, v = (torch.zeros(rows, kvh, 128, dtype=BF, device="cuda") for _ in range(2))
    out = tables.outputs(rows)
    new = torch.ones(rows, dtype=torch.int32, device="cuda")
    result = torch.zeros_like(q)

    def step():
        runner.prepare_decode_device(tables, new, out=out)
        result.copy_(layer(q, k, v).view(rows, heads, 128))

    graph = None
    if capture:
        state = [tables.context_lens, tables.num_blocks, tables.block_tables, tables.free_blocks,
                 tables.num_free, runner.kv_cache]
        saved = [x.clone() for x in state]
        step()
        torch.cuda.synchronize()
        for x, s in zip(state, saved):
            x.copy_(s)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            step()
    none = torch.zeros(0, kvh, 128, dtype=torch.float64)
    hist, waited = [(none, none)] * rows, 0
    for i in range(70):
        nq = torch.randn(rows, heads, 128, generator=gen).to(BF)
        nk, nv = (torch.randn(rows, kvh, 128, generator=gen).to(BF) for _ in range(2))
        q.copy_(nq), k.copy_(nk), v.copy_(nv)
        before = runner.kv_cache[:, :, :4].clone()
        graph.replay() if graph is not None else step()
        torch.cuda.synchronize()
        granted = out.query_lens.tolist()
        changed = (runner.kv_cache[:, 0, :4] != before[:, 0]).any(-1).any(-1)
        assert int(changed.sum()) == 2 * sum(granted)     # a token's K and V rows each
        for b in range(rows):
            if not granted[b]:
                waited += 1
                assert result[b].isnan().all()
                continue
            hist[b] = (torch.cat((hist[b][0], nk[b:b + 1].double())),
                       torch.cat((hist[b][1], nv[b:b + 1].double())))
            if i % 7 == 0:
                want, _ = fo.attend(nq[b:b + 1], *hist[b], fo.causal(1, len(hist[b][0])), SCALE)
                off = (result[b:b + 1].double().cpu() - want).abs()
                # (the paged decode's bar over a bf16 pool)
                assert float(off.max()) < 2e-2 and float(off.mean()) < 2e-3, (i, b)
    assert waited > 0


def test_blocks_travel_with_their_powers():
    """Codes and powers over the wire's staging, each as a pool: 4-bit blocks come out
    of another runner's blocks as they went in."""
    from nanovllm_amd.pd.kv_channel import LocalKVChannel
    here, _ = _runner(layers=2)
    there, _ = _runner(layers=2)
    gen = torch.Generator(device="cuda").manual_seed(7)
    for t in (here.kv_cache, here.kv_scales):
        t.copy_(torch.randint(0, 250, t.shape, dtype=torch.uint8, device="cuda", generator=gen))
    src, dst = [3, 0, 17], [5, 20, 1]
    for a, b in ((here.kv_cache, there.kv_cache), (here.kv_scales, there.kv_scales)):
        buf = LocalKVChannel(a).send(src)
        LocalKVChannel(b).recv(dst, buf)
        assert torch.equal(b[:, :, dst], a[:, :, src])
        rest = [i for i in range(25) if i not in dst]
        assert (b[:, :, rest] == (0 if b is there.kv_cache else 127)).all()


def test_captured_step_refuses_scales_of_another_pool():
    pool = torch.zeros(3, PAGE, KVH, 128, dtype=BF, device="cuda")
    scale = torch.zeros(3, PAGE, KVH, 4, dtype=torch.uint8, device="cuda")
    with pytest.raises(ValueError, match="4-bit"):
        DecodeGraphRunner([pool], [pool.clone()], HEADS, 2, 2, SCALE, k_scales=[scale],
                          v_scales=[scale])


@pytest.mark.parametrize("kind", ["tokhead", "chan"])
@pytest.mark.parametrize("capture", [False, True])
def test_serving_loop_over_an_int8_pool(kind, capture):
    """The same loop over the int8 pools: bit for bit the step whose slots, lengths and
    tables the host wrote, rows that wait among them (NaN, and the pool as it was)."""
    rows, kvh, heads, blocks, width = 3, 4, 8, 4, 3
    gen = torch.Generator().manual_seed(8)
    scales = (0.01 + 0.02 * torch.rand(kvh, 128, generator=gen)).cuda()
    sides = []
    for _ in range(2):
        runner = KVCacheRunner(1, blocks, PAGE, kvh, 128, kv_int8=kind)
        runner.kv_cache.zero_()
        if kind == "chan":
            runner.kv_scales.copy_(scales.expand_as(runner.kv_scales))
            runner.kv_dscales.copy_(runner.kv_scales)
        layer = Attention(heads, 128, SCALE, kvh)
        assert runner.bind([layer]) == 1
        sides.append((runner, layer))
    (runner, layer), (other, host_layer) = sides
    tables = runner.device_tables(rows, width)
    q = torch.zeros(rows, heads, 128, dtype=BF, device="cuda")
    k, v = (torch.zeros(rows, kvh, 128, dtype=BF, device="cuda") for _ in range(2))
    new = torch.ones(rows, dtype=torch.int32, device="cuda")
    out = tables.outputs(rows)
    result = torch.zeros_like(q)

    def step():
        runner.prepare_decode_device(tables, new, out=out)
        result.copy_(layer(q, k, v).view(rows, heads, 128))

    graph = None
    if capture:
        state = [tables.context_lens, tables.num_blocks, tables.block_tables, tables.free_blocks,
                 tables.num_free, runner.kv_cache, runner.kv_scales]
        saved = [x.clone() for x in state]
        step()
        torch.cuda.synchronize()
        for x, s in zip(state, saved):
            x.copy_(s)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            step()
    lens, mine = [0] * rows, [[] for _ in range(rows)]
    free, waited = list(range(blocks)), 0
    for i in range(70):
        nq = torch.randn(rows, heads, 128, generator=gen).to(BF)
        nk, nv = (torch.randn(rows, kvh, 128, generator=gen).to(BF) for _ in range(2))
        q.copy_(nq), k.copy_(nk), v.copy_(nv)
        graph.replay() if graph is not None else step()
        torch.cuda.synchronize()
        slots, seen = [], []
        for b in range(rows):                   # rows in order; pages off the stack's top
            if lens[b] == PAGE * len(mine[b]) and not free:
                slots.append(other.scratch_slot), seen.append(0)
                waited += 1
                continue
            if lens[b] == PAGE * len(mine[b]):
                mine[b].append(free.pop())
            slots.append(mine[b][lens[b] // PAGE] * PAGE + lens[b] % PAGE)
            lens[b] += 1
            seen.append(lens[b])
        set_context(False, slot_mapping=torch.tensor(slots, dtype=torch.int32).cuda(),
                    context_lens=torch.tensor(seen, dtype=torch.int32).cuda(),
                    block_tables=torch.tensor([m + [-1] * (width - len(m)) for m in mine],
                                              dtype=torch.int32).cuda(),
                    max_context_len=width * PAGE)
        want = host_layer(q, k, v).view(rows, heads, 128)
        for b in range(rows):
            if seen[b]:
                assert torch.equal(result[b], want[b]) and torch.isfinite(want[b]).all(), (i, b)
            else:
                assert result[b].isnan().all(), (i, b)
        assert torch.equal(runner.kv_cache[:, :, :blocks], other.kv_cache[:, :, :blocks]), i
        if kind == "tokhead":
            assert torch.equal(runner.kv_scales[:, :, :blocks], other.kv_scales[:, :, :blocks]), i
    assert waited > 0
