"""The device-built step tables against a row-by-row Python model, which hands out
pages and tokens in order; whole numbers, so everything is equal or wrong."""
import random

import pytest
import torch

from nanovllm_amd import _native
from nanovllm_amd.engine.device_tables import DeviceBlockTables
from nanovllm_amd.kernels.step_tables import (NO_SLOT, StepTables, build_step_tables,
                                              new_step_tables)

pytestmark = pytest.mark.gpu


def model(lens, new, table, held, free, num_free, page, tokens, per_row, finished, pad):
    """What build_step_tables says, on lists; tables and the stack change in place."""
    width = len(table[0]) if table else 0
    batch = len(lens)
    lens = [max(0, min(n, 1 << 29)) for n in lens]
    new = [max(0, min(n, 1 << 29)) for n in new]
    held = [max(0, min(n, width)) for n in held]
    top = max(0, min(num_free, len(free)))
    for b in range(batch):
        if finished[b]:
            for j in range(held[b]):
                if top < len(free):
                    free[top] = table[b][j]
                top += 1
            held[b] = lens[b] = 0
    top = min(top, len(free))
    need_sum = want_sum = taken = 0
    got, seen = [0] * batch, [0] * batch
    pool_top = top
    for b in range(batch):
        pages = (lens[b] + new[b] + page - 1) // page
        able = new[b] > 0 and pages <= width
        need = max(0, pages - held[b]) if able else 0
        need_sum += need
        able = able and (need == 0 or need_sum <= pool_top)
        want = new[b] if able else 0
        if per_row:
            able = able and want <= per_row
        else:
            want_sum += want
            able = able and want_sum <= tokens
        if able:
            got[b], seen[b] = new[b], lens[b] + new[b]
            for _ in range(need):
                table[b][held[b]] = free[pool_top - 1 - taken]
                held[b] += 1
                taken += 1
    slots, positions = [pad] * tokens, [0] * tokens
    at = 0
    cu_q, cu_k = [0], [0]
    for b in range(batch):
        first = b * per_row if per_row else at
        for i in range(got[b]):
            pos = lens[b] + i
            positions[first + i] = pos
            entry = table[b][pos // page]
            if entry >= 0 and entry * page + pos % page < 1 << 31:
                slots[first + i] = entry * page + pos % page
        at += got[b]
        cu_q.append(cu_q[-1] + got[b])
        cu_k.append(cu_k[-1] + seen[b])
    return dict(slot_mapping=slots, positions=positions, query_lens=got, seq_lens=seen,
                context_lens=[a + g for a, g in zip(lens, got)], cu_seqlens_q=cu_q,
                cu_seqlens_k=cu_k, num_blocks=held, num_free=[top - taken])


def _state(rng, batch, page, width, longest, free):
    lens = [rng.randint(0, min(longest, width * page)) for _ in range(batch)]
    held = [min(width, (n + page - 1) // page + (rng.random() < 0.2)) for n in lens]
    ids = list(range(sum(held) + free))
    rng.shuffle(ids)
    table, at = [], 0
    for h in held:
        table.append(ids[at:at + h] + [-1] * (width - h))
        at += h
    return lens, held, table, ids[at:] + [0] * sum(held), free


def _i32(x):
    return torch.tensor(x, dtype=torch.int32).cuda()


def _compare(lens, new, table, held, free, num_free, page, tokens, per_row=0, finished=None,
             pad=NO_SLOT, in_place=False, view=False, host=True):
    batch, width = len(table), len(table[0])
    if view:
        big = torch.full((batch, width + 5), 77, dtype=torch.int32).cuda()
        dev_table = big[:, 2:2 + width]
        dev_table.copy_(_i32(table))
    else:
        dev_table = _i32(table)
    dev = dict(lens=_i32(lens), new=_i32(new), held=_i32(held), free=_i32(free),
               num=_i32([num_free]))
    gone = None if finished is None else torch.tensor(finished).cuda()
    out = None
    if in_place:
        out = new_step_tables(batch, tokens, "cuda")
        out.num_blocks, out.num_free = dev["held"], dev["num"]
        out.context_lens, out.query_lens = dev["lens"], dev["new"]
    got = build_step_tables(dev["lens"], dev["new"], dev_table, dev["held"], dev["free"],
                            dev["num"], page, tokens, tokens_per_row=per_row, finished=gone,
                            pad_slot=pad, out=out)
    table, free = [list(r) for r in table], list(free)
    want = model(lens, new, table, held, free, num_free, page, tokens, per_row,
                 finished or [False] * batch, pad)
    assert isinstance(got, StepTables)
    for name, w in want.items():
        assert getattr(got, name).tolist() == w, name
    assert dev_table.tolist() == table, "block_tables"
    assert dev["free"].tolist() == free, "free_blocks"
    if view:
        assert (big[:, :2] == 77).all() and (big[:, 2 + width:] == 77).all()
    return want


@pytest.mark.parametrize("seed", range(40))
def test_against_the_model(seed):
    rng = random.Random(seed)
    batch = rng.choice([1, 2, 7, 63, 64, 65, 200])
    page = rng.choice([1, 16, 32, 48, 256])
    width = rng.randint(1, 12)
    lens, held, table, free, num = _state(rng, batch, page, width, width * page, rng.randint(0, 30))
    per_row = rng.choice([0, 0, 0, 1, 5])
    new = [rng.choice([0, 1, 1, 1, per_row or rng.randint(1, 3 * page)]) for _ in range(batch)]
    finished = [rng.random() < 0.2 for _ in range(batch)] if seed % 3 else None
    tokens = batch * per_row or max(1, int(sum(new) * rng.choice([0.5, 1, 1.2])) + 1)
    _compare(lens, new, table, held, free, num, page, tokens, per_row, finished,
             pad=rng.choice([NO_SLOT, -1, 12345]), in_place=seed % 2 == 0, view=seed % 5 == 0)


@pytest.mark.parametrize("batch,tokens", [(1024, 3000), (1025, 3000), (2500, 60000), (4096, 4096),
                                          (4097, 4200), (5000, 100)])
def test_many_rows_and_tokens(batch, tokens):
    """One and several rounds of rows, both ways to fill the tokens, offsets in and out
    of LDS, rows that no longer fit."""
    rng = random.Random(batch)
    lens, held, table, free, num = _state(rng, batch, 32, 6, 150, batch // 2)
    new = [rng.choice([0, 1, 1, rng.randint(1, 40)]) for _ in range(batch)]
    want = _compare(lens, new, table, held, free, num, 32, tokens,
                    finished=[rng.random() < 0.1 for _ in range(batch)])
    assert 0 < want["cu_seqlens_q"][-1] <= tokens


def test_long_prompts():
    """Rows that take many pages at once, more than a wave's lanes; tokens past one
    launch; a prompt too long for its table."""
    rng = random.Random(3)
    lens, held, table, free, num = _state(rng, 5, 16, 700, 500, 2500)
    _compare(lens, [9000, 1, 6001, 40000, 3], table, held, free, num, 16, 20000)


def test_pages_and_tokens_run_out():
    """The row that does not fit waits, and so do later ones that need a page; one that
    needs none goes on; after the step is full nobody does."""
    table = [[0, -1], [1, -1], [2, -1], [3, -1], [4, -1]]
    want = _compare([32, 32, 31, 32, 10], [1, 33, 1, 1, 4], table, [1] * 5, [9, 8], 2, 32, 64)
    # (the second row's 65 tokens are too wide for its table: it asks for no page)
    assert want["query_lens"] == [1, 0, 1, 1, 4] and want["num_free"] == [0]
    table = [r + [-1] for r in table]
    want = _compare([32, 32, 31, 32, 10], [1, 33, 1, 1, 4], table, [1] * 5, [9, 8], 2, 32, 64)
    assert want["query_lens"] == [1, 0, 1, 0, 4] and want["num_free"] == [1]
    want = _compare([1, 1, 1], [4, 5, 1], [[0], [1], [2]], [1] * 3, [7], 1, 32, 8)
    assert want["query_lens"] == [4, 0, 0]
    want = _compare([0], [1], [[-1]], [0], [], 0, 32, 1)
    assert want["query_lens"] == [0] and want["slot_mapping"] == [NO_SLOT]


def test_finished_rows_restart():
    """A row whose request ended takes a new one in the same step: its old pages go
    back first and are the first to be handed out."""
    table = [[5, 6, 7], [1, -1, -1]]
    want = _compare([90, 20], [40, 1], table, [3, 1], [2, 0, 0, 0, 0], 1, 32, 64,
                    finished=[True, False])
    assert want["num_blocks"] == [2, 1] and want["num_free"] == [2]
    # a stack without room drops what does not fit instead of writing past its end
    _compare([90], [0], [[5, 6, 7]], [3], [2, 0], 1, 32, 4, finished=[True])


def test_values_out_of_range():
    """Lengths, counts and table entries that no state holds: nothing is read or
    written outside the given tensors."""
    big = 2 ** 31 - 1
    _compare([-5, big, 3, 0], [2, 1, -7, big], [[0, 1], [2, 3], [4, -1], [-1, -1]],
             [-3, 9, 1, 0], [8, 9, 0], 3, 32, 16)
    _compare([3, 3], [1, 1], [[-9], [big]], [1, 1], [8], 99, 32, 4)
    _compare([3, 3], [1, 1], [[0], [1]], [1, 1], [8], -4, 32, 4)


def test_host_and_python_paths_agree(monkeypatch):
    rng = random.Random(8)
    args = _state(rng, 9, 32, 5, 100, 9)
    _compare(*[args[0], [1] * 9, *[args[2], args[1], args[3], args[4]]], 32, 9, 1)
    monkeypatch.setattr(_native, "_host", _native._NoHostPath)
    _compare(*[args[0], [1] * 9, *[args[2], args[1], args[3], args[4]]], 32, 9, 1)


@pytest.mark.parametrize("native", [True, False])
def test_outputs_are_apart(native, monkeypatch):
    """Fields of one result may share memory with nobody: each is written over and the
    others keep their values; they outlive the rest of the result."""
    if not native:
        monkeypatch.setattr(_native, "_host", _native._NoHostPath)
    names = ("slot_mapping", "positions", "query_lens", "seq_lens", "context_lens",
             "cu_seqlens_q", "cu_seqlens_k", "num_blocks", "num_free")
    for batch, tokens in ((1, 1), (5, 7), (17, 33)):
        table = torch.full((batch, 2), -1, dtype=torch.int32, device="cuda")
        zero = torch.zeros(batch, dtype=torch.int32, device="cuda")
        free = torch.arange(40, dtype=torch.int32, device="cuda")
        got = build_step_tables(zero, zero + 1, table, zero, free, _i32([40]), 32, tokens)
        before = {n: getattr(got, n).tolist() for n in names}
        assert [getattr(got, n).numel() for n in names] == [tokens, tokens, batch, batch, batch,
                                                            batch + 1, batch + 1, batch, 1]
        for i, n in enumerate(names):
            getattr(got, n).fill_(-100 - i)
            for other in names[i + 1:]:
                assert getattr(got, other).tolist() == before[other], (n, other)
        keep = got.num_free
        del got
        torch.empty(1 << 16, dtype=torch.int32, device="cuda").fill_(3)
        assert keep.tolist() == [-108] and keep.dtype == torch.int32


def test_under_inference_mode():
    """As a server runs: results are ordinary inference tensors, in place and as inputs
    of the next step."""
    with torch.inference_mode():
        t = DeviceBlockTables(3, 4, 16, 9)
        got = t.step(_i32([17, 1, 0]), 32)
        again = build_step_tables(got.context_lens, _i32([1, 1, 1]), t.block_tables,
                                  got.num_blocks, t.free_blocks, got.num_free, 16, 3,
                                  tokens_per_row=1)
        assert again.context_lens.tolist() == [18, 2, 1]
        assert again.positions.tolist() == [17, 1, 0]
        assert again.slot_mapping.is_inference() and again.positions.is_inference()
        again.slot_mapping.add_(1)
        kept = (again.positions + 1).clone()
    assert kept.tolist() == [18, 2, 1]
    again = build_step_tables(_i32([0]), _i32([1]), _i32([[-1]]), _i32([0]), _i32([5]), _i32([1]),
                              16, 1)
    assert not again.slot_mapping.is_inference() and again.slot_mapping.add_(1).tolist() == [81]


def test_empty_shapes():
    none = torch.zeros(0, dtype=torch.int32, device="cuda")
    num = _i32([3])
    got = build_step_tables(none, none, torch.zeros(0, 4, dtype=torch.int32, device="cuda"), none,
                            _i32([1, 2, 3]), num, 32, 5)
    assert got.slot_mapping.tolist() == [NO_SLOT] * 5 and got.positions.tolist() == [0] * 5
    assert got.cu_seqlens_q.tolist() == [0] == got.cu_seqlens_k.tolist()
    assert got.num_free.tolist() == [3]
    got = build_step_tables(_i32([4, 4]), _i32([1, 1]),
                            torch.zeros(2, 1, dtype=torch.int32, device="cuda"), _i32([1, 1]),
                            _i32([3]), num, 32, 0)
    assert got.query_lens.tolist() == [0, 0] and got.slot_mapping.numel() == 0


def test_state_over_steps_and_streams():
    """DeviceBlockTables over 40 steps of requests that come, grow, draft and go, on a
    stream of its own; the model keeps the same state."""
    rng = random.Random(12)
    rows, width, page, pages = 6, 8, 32, 30
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        t = DeviceBlockTables(rows, width, page, pages, pad_slot=pages * page)
        lens, held = [0] * rows, [0] * rows
        table, free, num = [[-1] * width for _ in range(rows)], list(range(pages)), pages
        out = t.outputs(64)
        for i in range(40):
            finished = [rng.random() < 0.1 for _ in range(rows)]
            new = [0 if f and rng.random() < 0.5 else rng.choice([1, 1, 8, 70]) for f in finished]
            got = t.step(_i32(new), 64, finished=torch.tensor(finished).cuda(),
                         out=out if i % 2 else None)
            want = model(lens, new, table, held, free, num, page, 64, 0, finished, pages * page)
            for name, w in want.items():
                assert getattr(got, name).tolist() == w, (i, name)
            assert t.block_tables.tolist() == table and t.free_blocks.tolist() == free
            lens, held, num = want["context_lens"], want["num_blocks"], want["num_free"][0]
            held_pages = [p for r, h in zip(table, held) for p in r[:h]]
            assert sorted(held_pages + free[:num]) == list(range(pages))   # none lost, none twice
            if i % 4 == 3:                                  # some drafts were not accepted
                lens = [max(0, n - rng.randint(0, 5)) for n in lens]
                t.context_lens.copy_(_i32(lens))
    stream.synchronize()


@pytest.mark.parametrize("tokens", [6, 5000])
def test_captured(tokens):
    """A captured step that advances its own state, replayed with eager steps between
    and requests that end."""
    rows, width, page = 6, 40, 16
    t = DeviceBlockTables(rows, width, page, 200)
    per_row = 1 if tokens == rows else 0
    new = _i32([1] * rows if per_row else [17, 0, 3, 1, 1, 20])
    finished = torch.zeros(rows, dtype=torch.bool, device="cuda")
    out = t.outputs(tokens)

    def step():
        t.step(new, tokens, tokens_per_row=per_row, finished=finished, out=out)

    state = [t.context_lens, t.num_blocks, t.block_tables, t.free_blocks, t.num_free]
    saved = [x.clone() for x in state]
    step()
    torch.cuda.synchronize()
    for x, s in zip(state, saved):
        x.copy_(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    lens, held = [0] * rows, [0] * rows
    table, free, num = [[-1] * width for _ in range(rows)], list(range(200)), 200
    for i in range(9):
        gone = [i == 5 and b == 2 for b in range(rows)]
        finished.copy_(torch.tensor(gone))
        if i % 3 == 2:
            step()
        else:
            graph.replay()
        torch.cuda.synchronize()
        want = model(lens, new.tolist(), table, held, free, num, page, tokens, per_row, gone,
                     NO_SLOT)
        for name, w in want.items():
            assert getattr(out, name).tolist() == w, (i, name)
        assert t.block_tables.tolist() == table and t.free_blocks.tolist() == free
        lens, held, num = want["context_lens"], want["num_blocks"], want["num_free"][0]


@pytest.mark.parametrize("capture", [False, True])
@pytest.mark.parametrize("marks", [torch.bool, torch.uint8])
def test_drafted_tokens_and_requests_that_end(capture, marks):
    """advance=False: a step grants drafts, of which some are accepted and added to the
    state by the caller.  A row whose request ended starts empty in the state too,
    whether or not a new one takes it in the same step."""
    rng = random.Random(21)
    rows, width, page, pages, tokens = 5, 6, 16, 24, 64
    t = DeviceBlockTables(rows, width, page, pages)
    new = torch.zeros(rows, dtype=torch.int32, device="cuda")
    finished = torch.zeros(rows, dtype=marks, device="cuda")
    out = t.outputs(tokens, advance=False) if capture else None

    def step():
        return t.step(new, tokens, finished=finished, advance=False, out=out)

    graph = None
    if capture:
        state = [t.context_lens, t.num_blocks, t.block_tables, t.free_blocks, t.num_free]
        saved = [x.clone() for x in state]
        step()
        torch.cuda.synchronize()
        for x, s in zip(state, saved):
            x.copy_(s)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            step()
    lens, held = [0] * rows, [0] * rows
    table, free, num = [[-1] * width for _ in range(rows)], list(range(pages)), pages
    ended = 0
    for i in range(40):
        gone = [rng.random() < 0.15 for _ in range(rows)]
        ended += sum(g and n > 0 for g, n in zip(gone, lens))
        asked = [rng.choice([0, 1, 4, 30]) for _ in range(rows)]
        new.copy_(_i32(asked))
        finished.copy_(torch.tensor(gone))
        if graph is None or i % 4 == 3:
            got = step()
        else:
            graph.replay()
            got = out
        torch.cuda.synchronize()
        want = model(lens, asked, table, held, free, num, page, tokens, 0, gone, NO_SLOT)
        for name, w in want.items():
            assert getattr(got, name).tolist() == w, (i, name)
        assert t.block_tables.tolist() == table and t.free_blocks.tolist() == free
        lens = [0 if g else n for g, n in zip(gone, lens)]
        assert t.context_lens.tolist() == lens, i
        held, num = want["num_blocks"], want["num_free"][0]
        accepted = [rng.randint(0, g) for g in want["query_lens"]]
        t.context_lens.add_(_i32(accepted))
        lens = [n + a for n, a in zip(lens, accepted)]
    assert ended > 5


def test_ended_lengths_of_the_state_alone():
    """clear_ended touches the lengths of rows that ended, and without it none."""
    for clear in (False, True):
        lens = _i32([40, 20, 7])
        build_step_tables(lens, _i32([1, 0, 1]), _i32([[0, 1], [2, 3], [4, -1]]), _i32([2, 2, 1]),
                          _i32([0] * 8), _i32([0]), 32, 4,
                          finished=torch.tensor([True, True, False]).cuda(),
                          clear_ended=clear)
        assert lens.tolist() == ([0, 0, 7] if clear else [40, 20, 7])
    lens = _i32([40])
    with pytest.raises(ValueError, match="ended"):
        out = new_step_tables(1, 4, "cuda")
        out.context_lens = lens
        build_step_tables(lens, _i32([1]), _i32([[0, 1]]), _i32([2]), _i32([0] * 4), _i32([0]), 32,
                          4, finished=torch.tensor([True]).cuda(), clear_ended=True, out=out)
    assert lens.tolist() == [40]


@pytest.mark.parametrize("batch", [700, 1500])
def test_wants_whose_sum_passes_32_bits(batch):
    """Rows that hold room for 2^22 tokens each and ask for all of it, 512 of which pass
    2^31: rows behind them wait as those do, however small their wish."""
    tokens = (1 << 22) - 1
    lens = [0] * batch
    held = [4] * batch
    table = [[b, b + 1, b + 2, b + 3] for b in range(batch)]
    new = [1 << 22] * batch
    new[0], new[batch - 100:] = 7, [3] * 100
    got = build_step_tables(_i32(lens), _i32(new), _i32(table), _i32(held), _i32([]), _i32([0]),
                            1 << 20, tokens)
    assert got.query_lens.tolist() == [7] + [0] * (batch - 1)
    want = model(lens, new, table, held, [], 0, 1 << 20, tokens, 0, [False] * batch, NO_SLOT)
    for name, w in want.items():
        equal = getattr(got, name).tolist() == w       # (lists too long to be shown apart)
        assert equal, name
