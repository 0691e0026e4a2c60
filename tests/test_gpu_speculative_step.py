"""The operators together, as a serving program runs them: an image prompt's
prefill (three-axis positions, two-way prefix, capped and windowed scores), a
step of drafted trees, the accepted path kept in every layer, and decoding on,
through the bound attention layers.  The same tokens decoded one by one give
the same cache bytes and, within the kernels' roundings, the same outputs."""
import pytest
import torch

from nanovllm_amd.engine.kv_runner import KVCacheRunner
from nanovllm_amd.kernels.tree import tree_mask_from_parents
from nanovllm_amd.layers.attention import Attention
from nanovllm_amd.layers.rotary import build_cos_sin_cache
from nanovllm_amd.utils.context import reset_context, set_context

pytestmark = pytest.mark.gpu
DEV = "cuda"
H, KVH, PAGE, LAYERS = 16, 2, 32, 3
SECTIONS = (24, 20, 20)
I32 = dict(dtype=torch.int32, device=DEV)


class _Model:
    """Attention layers over one pool; a token's qkv in a layer is a table row,
    so that the same token gives the same projection in any step."""

    def __init__(self, seed, **shape):
        gen = torch.Generator().manual_seed(seed)
        self.qkv = torch.randn(LAYERS, 200, (H + 2 * KVH) * 128, generator=gen) \
            .to(torch.bfloat16).to(DEV)
        self.w = [(1 + 0.1 * torch.randn(128, generator=gen)).to(torch.bfloat16).to(DEV)
                  for _ in range(2)]
        self.table = build_cos_sin_cache(128, 512, 1e4, DEV)
        self.layers = [Attention(H, 128, 128 ** -0.5, KVH, **shape) for _ in range(LAYERS)]
        self.kv = KVCacheRunner(LAYERS, 24, PAGE, KVH, 128, device=DEV)
        self.kv.kv_cache.fill_(float("nan"))
        assert self.kv.bind(self.layers) == LAYERS

    def forward(self, tokens, positions):
        outs = []
        for layer, attn in enumerate(self.layers):
            q, k, v = self.qkv[layer, tokens].split((H * 128, KVH * 128, KVH * 128), dim=-1)
            outs.append(attn.forward_fused(positions, q, k, v, self.table, self.w[0], self.w[1],
                                           1e-6, rope_sections=SECTIONS, rope_interleaved=True))
        return torch.stack(outs)


def _slots(tables, row, a, b):
    return [int(tables[row][p // PAGE]) * PAGE + p % PAGE for p in range(a, b)]


@pytest.mark.parametrize("shape", [dict(), dict(softcap=30.0), dict(window=20, softcap=50.0),
                                   dict(alibi=True)])
def test_prompt_draft_keep_decode(shape):
    shape = dict(shape)
    if shape.pop("alibi", False):
        shape["alibi_slopes"] = torch.tensor([2.0 ** -(i + 1) for i in range(H)], device=DEV)
    if not shape:
        shape = dict(softcap=0.0)
    prompts, images = [45, 70], [12, 40]
    tables = [[7, 3, 11, 0], [2, 9, 5, 14]]
    bt = torch.tensor(tables, **I32)
    parents = [[-1, 0, 0, 1, 2, 2, 5], [-1, 0, 1, 1, 3]]
    accepted = [[0, 2, 5, 6], [0, 1, 3]]
    gen = torch.Generator().manual_seed(5)
    prompt_tokens = [torch.randint(0, 200, (n,), generator=gen) for n in prompts]
    tree_tokens = [torch.randint(0, 200, (len(p),), generator=gen) for p in parents]
    after = torch.randint(0, 200, (2,), generator=gen)

    def place(n, image):
        """Image patches on a 4-wide grid, then text."""
        i = torch.arange(n)
        img = torch.stack((torch.zeros_like(i), i // 4, i % 4))
        text = (i - image + (image + 3) // 4).expand(3, -1)
        return torch.where(i < image, img, text)

    def prefill(model):
        cu = [0, prompts[0], sum(prompts)]
        set_context(True, torch.tensor(cu, **I32), torch.tensor(cu, **I32), max(prompts),
                    max(prompts),
                    torch.tensor(_slots(tables, 0, 0, prompts[0]) + _slots(tables, 1, 0, prompts[1]),
                                 **I32), None, bt, cu_seqlens_q_list=cu, cu_seqlens_k_list=cu,
                    prefix_lens=torch.tensor(images, **I32))
        pos = torch.cat([place(n, im) for n, im in zip(prompts, images)], dim=1).to(DEV)
        return model.forward(torch.cat(prompt_tokens).to(DEV), pos)

    def text_place(i, offset):
        return prompts[i] - images[i] + (images[i] + 3) // 4 + offset

    # One model drafts and keeps, the other decodes the accepted tokens one by one.
    a, b = _Model(3, **shape), _Model(3, **shape)
    assert torch.equal(prefill(a), prefill(b))

    sizes = [len(p) for p in parents]
    depth = [[0] * n for n in sizes]
    for i, p in enumerate(parents):
        for t, par in enumerate(p):
            depth[i][t] = depth[i][par] + 1 if par >= 0 else 0
    cu = [0, sizes[0], sum(sizes)]
    mask = tree_mask_from_parents(parents, DEV)
    set_context(False, torch.tensor(cu, **I32), None, max(sizes), 0,
                torch.tensor(sum((_slots(tables, i, prompts[i], prompts[i] + sizes[i])
                                  for i in range(2)), []), **I32),
                torch.tensor(prompts, **I32), bt, tree_mask=mask)
    pos = torch.tensor([text_place(i, d) for i in range(2) for d in depth[i]], device=DEV)
    drafted = a.forward(torch.cat(tree_tokens).to(DEV), pos.expand(3, -1))
    most = max(len(p) for p in accepted)
    a.kv.commit_tree(bt, torch.tensor(prompts, **I32),
                     torch.tensor([p + [-1] * (most - len(p)) for p in accepted], **I32),
                     torch.tensor([len(p) for p in accepted], **I32))

    for j in range(most):
        rows = [i for i in range(2) if j < len(accepted[i])]
        lens = [prompts[i] + j + 1 for i in rows]
        set_context(False, None, None, 0, 0,
                    torch.tensor([_slots(tables, i, n - 1, n)[0] for i, n in zip(rows, lens)], **I32),
                    torch.tensor(lens, **I32), bt[rows].contiguous(), max(lens))
        tok = torch.tensor([int(tree_tokens[i][accepted[i][j]]) for i in rows], device=DEV)
        pos = torch.tensor([text_place(i, j) for i in rows], device=DEV)
        out = b.forward(tok, pos.expand(3, -1))
        for r, i in enumerate(rows):
            want = out[:, r].float()
            got = drafted[:, cu[i] + accepted[i][j]].float()
            # two bf16 outputs of the same softmax: their weights' roundings
            # (2^-8 of |v - out|, |v| < 6 here) and their own
            assert float((got - want).abs().max()) <= 2 * 2.0 ** -8 * 12

    lens = [prompts[i] + len(accepted[i]) for i in range(2)]
    for i in range(2):
        at = torch.tensor(_slots(tables, i, 0, lens[i]), device=DEV)
        pa = a.kv.kv_cache.flatten(2, 3)[:, :, at]
        assert torch.equal(pa, b.kv.kv_cache.flatten(2, 3)[:, :, at])
        assert not torch.isnan(pa).any()

    set_context(False, None, None, 0, 0,
                torch.tensor([_slots(tables, i, lens[i], lens[i] + 1)[0] for i in range(2)], **I32),
                torch.tensor([n + 1 for n in lens], **I32), bt, max(lens) + 1)
    pos = torch.tensor([text_place(i, len(accepted[i])) for i in range(2)], device=DEV)
    nxt = [m.forward(after.to(DEV), pos.expand(3, -1)) for m in (a, b)]
    assert torch.equal(nxt[0], nxt[1])
    assert torch.isfinite(nxt[0].float()).all()
    reset_context()


def test_a_layer_over_an_int8_pool_refuses_shaped_scores():
    attn = Attention(H, 128, 0.1, KVH, softcap=30.0)
    attn.kv_cache_is_int8 = True
    set_context(False, context_lens=torch.ones(1, **I32))
    z = torch.zeros(1, H, 128, dtype=torch.bfloat16, device=DEV)
    with pytest.raises(ValueError, match="bf16 pool"):
        attn(z, z[:, :KVH], z[:, :KVH])
    reset_context()
