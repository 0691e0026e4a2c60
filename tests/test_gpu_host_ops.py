"""The native host path's shaped-score, tree, multi-axis rotary and commit
calls against the Python ones: the same bytes for every form it takes, the
Python path for every other form, the same refusals."""
import pytest
import torch

from nanovllm_amd import _native as nat
from nanovllm_amd.kernels.scored import scored_attention
from nanovllm_amd.kernels.tree import commit_tree_path, tree_attention, tree_mask_from_parents
from nanovllm_amd.layers.rotary import build_cos_sin_cache, qk_norm_mrope_store

pytestmark = pytest.mark.gpu
DEV = "cuda"
I32 = dict(dtype=torch.int32, device=DEV)
NAMES = ("scored", "tree", "mrope", "commit")


class _Sub(torch.Tensor):
    pass


def _both(monkeypatch, fn):
    """fn with the native path and without: (results or exception types,
    whether the native path served)."""
    real, served = nat.host(), []

    class Spy:
        pass

    for name in NAMES:
        def call(*a, f=getattr(real, name)):
            r = f(*a)
            served.append(r is not None)
            return r
        setattr(Spy, name, staticmethod(call))
    out = []
    for host in (Spy, nat._NoHostPath):
        monkeypatch.setattr(nat, "host", lambda h=host: h)
        try:
            out.append(fn())
        except Exception as e:  # noqa: BLE001
            out.append(type(e))
    monkeypatch.undo()
    torch.cuda.synchronize()
    return out, served[-1] if served else False


def _same(a, b):
    if isinstance(a, (tuple, list)):
        return all(_same(x, y) for x, y in zip(a, b))
    return torch.equal(a, b) if isinstance(a, torch.Tensor) else a == b


def _bf(*shape, seed=0):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    return torch.randn(*shape, generator=gen, device=DEV, dtype=torch.bfloat16)


def _pool():
    return _bf(9, 32, 2, 128, seed=1), _bf(9, 32, 2, 128, seed=2)


def _scored(**kw):
    kc, vc = _pool()
    args = dict(scale=0.1, block_tables=torch.arange(8, **I32).view(4, 2), num_decode_rows=2,
                decode_context_lens=torch.tensor([40, 9], **I32),
                cu_seqlens_q=torch.tensor([0, 3, 8], **I32),
                cu_seqlens_k=torch.tensor([0, 30, 64], **I32), cu_seqlens_q_list=[0, 3, 8],
                cu_seqlens_k_list=[0, 30, 64], softcap=30.0)
    args.update(kw)
    return scored_attention(args.pop("q", _bf(10, 8, 128, seed=3)), args.pop("kc", kc),
                            args.pop("vc", vc), **args)


def _fresh(**kw):
    return _scored(**{**dict(q=_bf(8, 8, 128, seed=4), kc=None, vc=None, block_tables=None,
                             num_decode_rows=0, decode_context_lens=None,
                             cu_seqlens_k=torch.tensor([0, 3, 8], **I32),
                             cu_seqlens_k_list=[0, 3, 8], k=_bf(8, 2, 128, seed=5),
                             v=_bf(8, 2, 128, seed=6)), **kw})


def _tree(**kw):
    kc, vc = _pool()
    args = dict(q=_bf(6, 8, 128, seed=7), block_tables=torch.arange(4, **I32).view(2, 2),
                context_lens=torch.tensor([40, 9], **I32),
                tree_mask=tree_mask_from_parents([[-1, 0, 0, 1], [-1, 0]], DEV), scale=0.1,
                cu_seqlens_q=torch.tensor([0, 4, 6], **I32), max_seqlen_q=4)
    args.update(kw)
    lead = [args.pop("q"), kc, vc] + [args.pop(n) for n in ("block_tables", "context_lens",
                                                            "tree_mask", "scale")]
    return tree_attention(*lead, **args)


def _mrope(**kw):
    kc, vc = _pool()
    args = dict(q=_bf(5, 8, 128, seed=8), k=_bf(5, 2, 128, seed=9), v=_bf(5, 2, 128, seed=10),
                positions=torch.arange(15, device=DEV).view(3, 5),
                cos_sin_cache=build_cos_sin_cache(128, 50, 1e4, DEV), sections=(24, 20, 20),
                interleaved=True, q_norm_weight=_bf(128, seed=11),
                k_norm_weight=_bf(128, seed=12), k_cache=kc, v_cache=vc,
                slot_mapping=torch.arange(5, **I32))
    args.update(kw)
    return [*qk_norm_mrope_store(**args), kc, vc]


def _commit(**kw):
    pool = torch.arange(2 * 3 * 6 * 4 * 16, device=DEV, dtype=torch.float32).view(2, 3, 6, 4, 16)
    args = dict(block_tables=torch.arange(6, **I32).view(2, 3),
                context_lens=torch.tensor([3, 5], **I32),
                paths=torch.tensor([[0, 2, 5], [1, 4, -1]], **I32),
                path_lens=torch.tensor([3, 2], **I32))
    args.update(kw)
    commit_tree_path(args.pop("pool", pool), *args.values())
    return pool


SERVED = [
    _scored, _fresh, _tree, _mrope, _commit,
    lambda: _scored(prefix_lens=torch.tensor([5, 0], **I32), window=7,
                    alibi_slopes=torch.rand(8, device=DEV, generator=torch.Generator(
                        device=DEV).manual_seed(1))),
    lambda: _scored(q=_bf(2, 8, 128), cu_seqlens_q=None, cu_seqlens_k=None,
                    cu_seqlens_q_list=None, cu_seqlens_k_list=None),
    lambda: _tree(cu_seqlens_q=None, max_seqlen_q=None, softcap=50.0, window=3,
                  tree_mask=tree_mask_from_parents([[-1, 0, 0], [-1, 0, 1]], DEV)),
    lambda: _mrope(return_k=False, q_norm_weight=None, v=None, k_cache=None, v_cache=None,
                   slot_mapping=None),
]
OTHERS = [     # taken by the Python path
    lambda: _scored(q=_bf(10, 8, 256)[..., ::2]),
    lambda: _scored(decode_context_lens=torch.tensor([40, 9], device=DEV)),
    lambda: _scored(softcap=30), lambda: _scored(scale=1), lambda: _scored(cu_seqlens_q=None),
    lambda: _scored(q=_bf(10, 8, 128, seed=3).as_subclass(_Sub)).as_subclass(torch.Tensor),
    lambda: _scored(cu_seqlens_q_list=(0, 3, 8)),
    lambda: _scored(block_tables=torch.arange(8, device=DEV).view(4, 2)),
    lambda: _tree(context_lens=torch.tensor([40, 9], device=DEV)),
    lambda: _tree(tree_mask=torch.ones(6, 2, dtype=torch.int64, device=DEV)[:, :1]),
    lambda: _mrope(q_out=torch.zeros(5, 8, 128, dtype=torch.bfloat16, device=DEV)),
    lambda: _mrope(positions=torch.arange(15, device=DEV).view(5, 3).t()),
    lambda: _mrope(q_norm_weight=torch.ones(128, device=DEV)),
    lambda: _commit(paths=torch.tensor([[0, 2, 5], [1, 4, -1]], device=DEV)),
]
REFUSED = [
    lambda: _scored(scale=-1.0), lambda: _scored(softcap=-1.0), lambda: _scored(window=-1),
    lambda: _scored(cu_seqlens_q_list=[0, 3, 7]), lambda: _scored(num_decode_rows=11),
    lambda: _scored(cu_seqlens_k_list=[0, 2, 64]), lambda: _scored(num_decode_rows=-1),
    lambda: _scored(block_tables=torch.zeros(3, 2, **I32)),
    lambda: _fresh(k=_bf(7, 2, 128)), lambda: _fresh(k=_bf(8, 3, 128), v=_bf(8, 3, 128)),
    lambda: _tree(max_seqlen_q=65), lambda: _tree(scale=float("inf")),
    lambda: _tree(cu_seqlens_q=torch.tensor([0, 4], **I32)), lambda: _tree(max_seqlen_q=None),
    lambda: _tree(tree_mask=torch.ones(5, 1, dtype=torch.int64, device=DEV)),
    lambda: _mrope(sections=(64, 1)), lambda: _mrope(positions=torch.zeros(2, 5, device=DEV)),
    lambda: _mrope(k_cache=_bf(9, 32, 3, 128), v_cache=_bf(9, 32, 3, 128)),
    lambda: _commit(paths=torch.zeros(3, 2, **I32)),
    lambda: _commit(pool=torch.zeros(2, 3, 4, device=DEV)),
]


@pytest.mark.parametrize("case", range(len(SERVED)))
def test_served_calls_give_the_same_bytes(monkeypatch, case):
    (a, b), served = _both(monkeypatch, SERVED[case])
    assert served and not isinstance(b, type) and _same(a, b)


@pytest.mark.parametrize("case", range(len(OTHERS)))
def test_other_forms_go_to_the_python_path(monkeypatch, case):
    (a, b), served = _both(monkeypatch, OTHERS[case])
    assert not served and not isinstance(b, type) and _same(a, b)


@pytest.mark.parametrize("case", range(len(REFUSED)))
def test_refusals_are_the_same(monkeypatch, case):
    (a, b), _ = _both(monkeypatch, REFUSED[case])
    assert isinstance(a, type) and a is b


def test_mrope_refuses_a_v_pool_alone(monkeypatch):
    """Without the k pool nothing would be appended."""
    (a, b), served = _both(monkeypatch, lambda: _mrope(k_cache=None))
    assert not served and a is b is ValueError
