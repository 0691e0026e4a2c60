"""Shaped attention layers in the contexts that the runner prepares: fresh
prompts without tables, a decode step, and a mixed step whose chunk goes on
over cached keys; every output against 64 bits over the tokens' own rows, and
the rows in the pool."""
import pytest
import torch

from nanovllm_amd.engine.kv_runner import KVCacheRunner
from nanovllm_amd.engine.sequence import Sequence
from nanovllm_amd.layers.attention import Attention
from nanovllm_amd.utils.context import get_context, reset_context
from scored_oracle import attend, check, chunk_mask, slopes_of

pytestmark = pytest.mark.gpu
DEV = "cuda"
H, KVH, PAGE = 16, 2, 32
SCALE = 128 ** -0.5


class _Step:
    """One layer over a pool, its sequences' rows kept beside it."""

    def __init__(self, monkeypatch, **shape):
        monkeypatch.setattr(Sequence, "block_size", PAGE)
        self.gen = torch.Generator().manual_seed(1)
        self.kv = KVCacheRunner(1, 20, PAGE, KVH, 128, device=DEV)
        self.kv.kv_cache.fill_(float("nan"))
        self.layer = Attention(H, 128, SCALE, KVH, **shape).to(DEV)
        self.kv.bind([self.layer])
        self.rows = {}

    def sequence(self, tokens, blocks):
        """(a decode step appends to the table's last block)"""
        seq = Sequence(range(tokens))
        seq.block_table = list(blocks)
        self.rows[seq.seq_id] = [torch.empty(0, KVH, 128, dtype=torch.bfloat16)
                                  for _ in range(2)]
        return seq

    def schedule(self, seq, cached, tokens):
        seq.num_cached_tokens, seq.num_scheduled_tokens = cached, tokens
        seq.is_prefill = tokens > 1 or cached == 0

    def run(self, seqs, label, prefix=None):
        """The step that the context describes; seqs in its row order."""
        sizes = [seq.num_scheduled_tokens for seq in seqs]
        n = sum(sizes)
        q, k, v = (torch.randn(n, h, 128, generator=self.gen).to(torch.bfloat16)
                   for h in (H, KVH, KVH))
        out = self.layer(q.to(DEV), k.to(DEV), v.to(DEV))
        torch.cuda.synchronize()
        at, layer = 0, self.layer
        sl = None if layer.alibi_slopes is None else layer.alibi_slopes.cpu()
        for i, (seq, size) in enumerate(zip(seqs, sizes)):
            rows = self.rows[seq.seq_id]
            for x, new in enumerate((k, v)):
                rows[x] = torch.cat((rows[x], new[at:at + size]))
            m = rows[0].size(0)
            pos = torch.arange(m)
            slot = torch.tensor(seq.block_table)[pos // PAGE] * PAGE + pos % PAGE
            for x in range(2):
                pool = self.kv.kv_cache[x, 0].flatten(0, 1)[slot.to(DEV)].cpu()
                assert torch.equal(pool, rows[x])
            w, b = attend(q[at:at + size], *rows,
                          *chunk_mask(size, m, layer.window, prefix[i] if prefix else 0),
                          scale=SCALE, cap=layer.softcap, slopes=sl)
            check(out[at:at + size], w, b, f"{label}, sequence {i}")
            at += size


@pytest.mark.parametrize("shape", [dict(softcap=30.0), dict(window=20, softcap=50.0),
                                   dict(alibi_slopes=slopes_of(H)), dict(window=33)])
@pytest.mark.parametrize("images", [False, True])
def test_prompts_decode_and_a_mixed_step(monkeypatch, shape, images):
    step = _Step(monkeypatch, **shape)
    a, b, c = (step.sequence(45, [4, 0]), step.sequence(70, [2, 7, 5]),
               step.sequence(90, [3, 11, 12]))

    # fresh prompts: no tables, the keys are the step's own
    step.schedule(a, 0, 45)
    step.schedule(b, 0, 70)
    step.kv.prepare_prefill([a, b])
    assert get_context().block_tables is None
    prefix = [12, 40] if images else None
    if images:
        get_context().prefix_lens = torch.tensor(prefix, dtype=torch.int32, device=DEV)
    step.run([a, b], "fresh", prefix)

    # one token each
    for seq in (a, b):
        seq.append_token(7)
        step.schedule(seq, len(seq) - 1, 1)
    step.kv.prepare_decode([a, b])
    step.run([a, b], "decode")

    # the first part of a third prompt, then decode rows beside its second
    step.schedule(c, 0, 50)
    step.kv.prepare_prefill([c])
    step.run([c], "first chunk")
    for seq in (a, b):
        seq.append_token(8)
        step.schedule(seq, len(seq) - 1, 1)
    step.schedule(c, 50, 40)
    step.kv.prepare_mixed([a, b, c])
    assert get_context().is_mixed and get_context().num_decode_rows == 2
    prefix = [0, 0, 60] if images else None
    if images:
        get_context().prefix_lens = torch.tensor(prefix[2:], dtype=torch.int32, device=DEV)
    step.run([a, b, c], "mixed", prefix)

    # a mixed step without chunks
    for seq in (a, b):
        seq.append_token(9)
        step.schedule(seq, len(seq) - 1, 1)
    step.kv.prepare_mixed([a, b])
    step.run([a, b], "mixed without chunks")
    reset_context()
