"""The captured decode step with shaped scores: every replay against the same
padded batch run eagerly (bit for bit: the same launches) and against 64 bits,
with eager work and synchronisations between the replays."""
import pytest
import torch

from nanovllm_amd.engine.graph_runner import DecodeGraphRunner, pad_decode_inputs
from nanovllm_amd.engine.kv_runner import KVCacheRunner
from nanovllm_amd.kernels.scored import scored_attention
from nanovllm_amd.layers.attention import Attention, store_kvcache
from nanovllm_amd.utils.context import reset_context, set_context
from scored_oracle import attend, check, chunk_mask, slopes_of

pytestmark = pytest.mark.gpu
DEV = "cuda"
LAYERS, HEADS, KVH, PAGE, BLOCKS, WIDTH = 3, 16, 2, 64, 40, 20
SCALE = 128 ** -0.5


def _batch(bs, seed):
    gen = torch.Generator().manual_seed(seed)
    lens = torch.randint(1, 1 + WIDTH * PAGE // max(1, bs - 1), (bs,), generator=gen).tolist()
    order = torch.randperm(BLOCKS, generator=gen).tolist()
    tables = torch.full((bs, WIDTH), -1, dtype=torch.int32)
    for i, n in enumerate(lens):
        need = (n + PAGE - 1) // PAGE
        tables[i, :need] = torch.tensor(order[:need], dtype=torch.int32)
        order = order[need:]
    slots = torch.tensor([int(tables[i, (n - 1) // PAGE]) * PAGE + (n - 1) % PAGE
                          for i, n in enumerate(lens)], dtype=torch.int32)
    q, k, v = (torch.randn(LAYERS, bs, h, 128, generator=gen).to(torch.bfloat16)
               for h in (HEADS, KVH, KVH))
    return q, k, v, slots, torch.tensor(lens, dtype=torch.int32), tables, lens


def test_replays_equal_the_eager_step():
    gen = torch.Generator().manual_seed(0)
    pools = [torch.randn(2, BLOCKS + 1, PAGE, KVH, 128, generator=gen).to(torch.bfloat16).to(DEV)
             for _ in range(LAYERS)]
    shapes = [dict(softcap=50.0, window=100), None,
              dict(alibi_slopes=slopes_of(HEADS).to(DEV))]
    runner = DecodeGraphRunner([p[0] for p in pools], [p[1] for p in pools], HEADS, max_bs=8,
                               max_blocks_per_seq=WIDTH, scale=SCALE, score_shapes=shapes)
    runner.capture()
    for rnd, bs in enumerate([3, 8, 1, 3, 5]):
        q, k, v, slots, lens, tables, host_lens = _batch(bs, 50 + rnd)
        b = runner.bucket_of(bs)
        sb = torch.empty(b, dtype=torch.int32, device=DEV)
        lb, tb = torch.empty_like(sb), torch.empty(b, WIDTH, dtype=torch.int32, device=DEV)
        pad_decode_inputs(slots.to(DEV), lens.to(DEV), tables.to(DEV), sb, lb, tb,
                          runner.scratch_slot, runner.scratch_block_id)
        copies = [p.clone() for p in pools]
        got = runner.run(q.to(DEV), k.to(DEV), v.to(DEV), slots.to(DEV), lens.to(DEV),
                         tables.to(DEV)).clone()
        torch.cuda.synchronize()
        for layer in (0, 2):
            kp = torch.zeros(b, KVH, 128, dtype=torch.bfloat16, device=DEV)
            vp = torch.zeros_like(kp)
            qp = torch.zeros(b, HEADS, 128, dtype=torch.bfloat16, device=DEV)
            kp[:bs], vp[:bs], qp[:bs] = k[layer].to(DEV), v[layer].to(DEV), q[layer].to(DEV)
            kc, vc = copies[layer][0], copies[layer][1]
            store_kvcache(kp, vp, kc, vc, sb)
            want = scored_attention(qp, kc, vc, scale=SCALE, block_tables=tb, num_decode_rows=b,
                                    decode_context_lens=lb, **shapes[layer])[:bs]
            assert torch.equal(got[layer].view(torch.int16), want.view(torch.int16))
            assert torch.equal(pools[layer].view(torch.int16), copies[layer].view(torch.int16))
            shape = dict(shapes[layer])
            sl = shape.pop("alibi_slopes", None)
            for i, n in enumerate(host_lens):
                pages = tables[i, :(n + PAGE - 1) // PAGE].long()
                ks, vs = (c.cpu()[pages].flatten(0, 1)[:n] for c in (kc, vc))
                w, bound = attend(q[layer, i:i + 1], ks, vs,
                                  *chunk_mask(1, n, shape.get("window", 0), 0), scale=SCALE,
                                  cap=shape.get("softcap", 0.0),
                                  slopes=None if sl is None else sl.cpu())
                check(got[layer, i:i + 1], w, bound, f"replay {rnd} layer {layer} row {i}")


def test_out_is_written_in_place():
    kc = torch.randn(4, 32, 2, 128, device=DEV).to(torch.bfloat16)
    q = torch.randn(2, 8, 128, device=DEV).to(torch.bfloat16)
    tables = torch.tensor([[0, 1], [2, 3]], dtype=torch.int32, device=DEV)
    lens = torch.tensor([40, 64], dtype=torch.int32, device=DEV)
    kw = dict(scale=SCALE, block_tables=tables, num_decode_rows=2, decode_context_lens=lens)
    want = scored_attention(q, kc, kc, **kw)
    wide = torch.full((2, 3, 8, 128), 7.0, dtype=torch.bfloat16, device=DEV)
    out = wide[:, 1]
    assert scored_attention(q, kc, kc, out=out, **kw) is out
    assert torch.equal(out, want)
    assert bool((wide[:, 0] == 7).all()) and bool((wide[:, 2] == 7).all())


def test_bound_layers_replay_as_they_run():
    """The captured step of a runner's bound layers, shaped or not, gives what
    the layers give eagerly, without their shapes being passed."""
    gen = torch.Generator().manual_seed(7)
    layers = [Attention(HEADS, 128, SCALE, KVH, softcap=30.0), Attention(HEADS, 128, SCALE, KVH),
              Attention(HEADS, 128, SCALE, KVH, alibi_slopes=slopes_of(HEADS), window=40).to(DEV)]
    kv = KVCacheRunner(LAYERS, BLOCKS, PAGE, KVH, 128, device=DEV)
    kv.kv_cache.copy_(torch.randn(kv.kv_cache.shape, generator=gen))
    kv.bind(layers)
    runner = DecodeGraphRunner.from_kv_runner(kv, HEADS, max_bs=4, max_blocks_per_seq=WIDTH,
                                              scale=SCALE)
    before = kv.kv_cache.clone()
    runner.capture()
    kv.kv_cache.copy_(before)
    for rnd in range(3):
        q, k, v, slots, lens, tables, host_lens = _batch(4, 70 + rnd)
        q, k, v, slots, lens, tables = (x.to(DEV) for x in (q, k, v, slots, lens, tables))
        got = runner.run(q, k, v, slots, lens, tables).clone()
        set_context(False, slot_mapping=slots, context_lens=lens, block_tables=tables,
                    max_context_len=max(host_lens))
        want = [layer(q[i], k[i], v[i]) for i, layer in enumerate(layers)]
        torch.cuda.synchronize()
        for i in (0, 2):
            # (a full bucket and tables of the same width: the same launches,
            # whose sums no timing orders)
            pages = [tables[r, :(n + PAGE - 1) // PAGE].long() for r, n in enumerate(host_lens)]
            for r, n in enumerate(host_lens):
                ks, vs = (kv.kv_cache[x, i][pages[r]].flatten(0, 1)[:n].cpu() for x in range(2))
                cap, window = layers[i].softcap, layers[i].window
                sl = layers[i].alibi_slopes
                w, b = attend(q[i, r:r + 1].cpu(), ks, vs, *chunk_mask(1, n, window, 0),
                              scale=SCALE, cap=cap, slopes=None if sl is None else sl.cpu())
                check(got[i, r:r + 1], w, b, f"round {rnd} layer {i} row {r}")
            assert torch.equal(got[i].view(torch.int16), want[i].view(torch.int16))
    reset_context()
