"""Accepted paths moved to the end of their contexts (kvc_commit_rows): byte
for byte, everything else untouched."""
import random

import pytest
import torch

from nanovllm_amd.engine.kv_runner import KVCacheRunner
from nanovllm_amd.kernels.tree import commit_tree_path

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _case(shape, page, ctx, room, seed):
    """A pool of `shape` = (planes.., blocks, page, ...) bytes and tables."""
    gen = torch.Generator().manual_seed(seed)
    need = [(c + room + page - 1) // page for c in ctx]
    order = torch.randperm(sum(need), generator=gen).to(torch.int32)
    tables = torch.full((len(ctx), max(need)), -1, dtype=torch.int32)
    at = 0
    for i, n in enumerate(need):
        tables[i, :n] = order[at:at + n]
        at += n
    return tables, sum(need)


def _want(pool, page, tables, ctx, paths, lens):
    out = pool.clone()
    flat, src = out.flatten(2, 3), pool.flatten(2, 3)
    for b, c in enumerate(ctx):
        last = -1
        for j in range(min(lens[b], paths.shape[1])):
            p = int(paths[b, j])
            if p <= last:
                break
            last = p
            s, d = c + p, c + j
            if s // page >= tables.shape[1] or int(tables[b, s // page]) < 0:
                break
            flat[:, :, int(tables[b, d // page]) * page + d % page] = \
                src[:, :, int(tables[b, s // page]) * page + s % page]
    return out


def _run(pool, page, tables, ctx, paths, lens):
    paths = torch.as_tensor(paths, dtype=torch.int32)
    want = _want(pool, page, tables, ctx, paths, lens)
    got = pool.to(DEV)
    commit_tree_path(got, tables.to(DEV), torch.tensor(ctx, dtype=torch.int32, device=DEV),
                     paths.to(DEV), torch.tensor(lens, dtype=torch.int32, device=DEV))
    torch.cuda.synchronize()
    assert torch.equal(got.cpu(), want)


@pytest.mark.parametrize("row,dtype", [((4, 128), torch.int16), ((3, 128), torch.int8),
                                       ((8, 128), torch.int16), ((4,), torch.float32),
                                       ((3,), torch.float32), ((2, 1), torch.int16),
                                       ((1, 3), torch.int8)])
@pytest.mark.parametrize("page", [32, 256])
def test_paths(row, dtype, page):
    rng = random.Random(len(row) + page)
    ctx = [0, 1, page - 1, page, 3 * page - 5, 77]
    room, most = 150, 100
    tables, blocks = _case(row, page, ctx, room, page)
    gen = torch.Generator().manual_seed(2)
    pool = torch.randint(-100, 100, (2, 3, blocks, page) + row, generator=gen).to(dtype)
    paths, lens = [], []
    for n in (0, 1, 3, 9, 64, 100):
        paths.append(sorted(rng.sample(range(room), n)) + [0] * (most - n))
        lens.append(n)
    _run(pool, page, tables, ctx, paths, lens)


def test_paths_end_where_they_stop_making_sense():
    page, ctx = 32, [10, 10, 10, 10, 10, 40]
    tables, blocks = _case((4, 128), page, ctx, 60, 5)
    pool = torch.randint(-100, 100, (2, 2, blocks, page, 2, 128)).to(torch.int16)
    tables[5, 2] = -1                       # its tree's last block is gone
    _run(pool, page, tables, ctx,
         [[0, 5, 5, 6], [3, 2, 7, 9], [-1, 0, 1, 2], [0, 1, 2, 3], [2, 1000000, 3, 4],
          [1, 9, 30, 31]], [4, 4, 4, 9, 4, 4])
    _run(pool, page, tables, ctx, [[0, 5, 5, 6]] * 6, [-3, 0, 2, 4, 1, 2])


def test_offsets_past_32_bits():
    """A plane of 4.6 GB: its last block takes part."""
    blocks, page = 4400, 256
    pool = torch.zeros(1, 1, blocks, page, 4, 128, dtype=torch.float16, device=DEV)
    pool[0, 0, blocks - 1] = torch.randn(page, 4, 128, device=DEV).half()
    want = pool[0, 0, blocks - 1].clone()
    want[100], want[101], want[102] = want[103].clone(), want[140].clone(), want[255].clone()
    commit_tree_path(pool, torch.tensor([[blocks - 1]], dtype=torch.int32, device=DEV),
                     torch.tensor([100], dtype=torch.int32, device=DEV),
                     torch.tensor([[3, 40, 155]], dtype=torch.int32, device=DEV),
                     torch.tensor([3], dtype=torch.int32, device=DEV))
    assert torch.equal(pool[0, 0, blocks - 1], want)
    assert float(pool[0, 0, :blocks - 1].abs().max()) == 0


@pytest.mark.parametrize("mode", [None, "tokhead", "chan"])
def test_runner_moves_everything_that_travels_with_a_row(mode):
    kv = KVCacheRunner(2, 5, 32, 2, 128, device=DEV, kv_int8=mode)
    pools = [p for p in (kv.kv_cache, kv.kv_side, kv.kv_scales if mode == "tokhead" else None)
             if p is not None]
    before = []
    for p in pools:
        p.copy_(torch.randint(-100, 100, p.shape, device=DEV).to(p.dtype))
        before.append(p.cpu().clone())
    tables = torch.tensor([[4, 0], [2, -1]], dtype=torch.int32)
    paths = torch.tensor([[0, 2, 9, 20], [1, 3, 0, 0]], dtype=torch.int32)
    lens, ctx = [4, 2], [20, 5]
    i32 = dict(dtype=torch.int32, device=DEV)
    kv.commit_tree(tables.to(DEV), torch.tensor(ctx, **i32), paths.to(DEV),
                   torch.tensor(lens, **i32))
    torch.cuda.synchronize()
    for p, was in zip(pools, before):
        assert torch.equal(p.cpu(), _want(was, 32, tables, ctx, paths, lens))


def test_captured_and_replayed():
    """One captured move serves other contexts, tables and paths, with eager
    moves between the replays."""
    page, room, most = 32, 40, 12
    tables, blocks = _case((2, 128), page, [60, 60], room, 7)
    gen = torch.Generator().manual_seed(8)
    pool = torch.randint(-100, 100, (2, 2, blocks, page, 2, 128), generator=gen).to(torch.int16)
    pool_d, table_d = torch.empty_like(pool, device=DEV), tables.to(DEV)
    i32 = dict(dtype=torch.int32, device=DEV)
    ctx_d, path_d, len_d = torch.zeros(2, **i32), torch.zeros(2, most, **i32), torch.zeros(2, **i32)

    def call():
        commit_tree_path(pool_d, table_d, ctx_d, path_d, len_d)

    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    rng = random.Random(9)
    for ctx in ([60, 3], [0, 31], [33, 64], [60, 3]):
        lens = [rng.randint(0, most) for _ in ctx]
        paths = torch.tensor([sorted(rng.sample(range(room - 8), n)) + [0] * (most - n)
                              for n in lens], dtype=torch.int32)
        table = tables.flip(0) if ctx[0] == 0 else tables
        ctx_d.copy_(torch.tensor(ctx, dtype=torch.int32))
        path_d.copy_(paths)
        len_d.copy_(torch.tensor(lens, dtype=torch.int32))
        table_d.copy_(table)
        want = _want(pool, page, table, ctx, paths, lens)
        for run in (graph.replay, call):
            pool_d.copy_(pool)
            run()
            torch.cuda.synchronize()
            assert torch.equal(pool_d.cpu(), want)
