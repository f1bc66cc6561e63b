"""A step's tables on the GPU against the same built request by request on the host:
every output equal, the tables behind it too; pages off the free list, a list that
is too short, padded steps, requests without tokens, rows outside the tables, more
requests and tokens than one round holds; captured and replayed."""

import pytest
import torch

from tinyserver_amd.kernels import step_tables

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _ints(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def _host(tables, rows, ctx, new, page, num_tokens, width, free):
    """The same, in lists. free: None or the list's entries."""
    tables = [list(t) for t in tables]
    w = len(tables[0]) if tables else 0
    taken, out, cu, pos, blk, slot = 0, [], [0], [], [], []
    for r, c, n in zip(rows, ctx, new):
        c, n = max(0, c), max(0, n)
        need = min(w, -(-(c + n) // page))
        have = min(w, -(-c // page)) if free is not None else need
        known = 0 <= r < len(tables)
        entries = list(tables[r][:need]) if known else [-1] * need
        if known:
            for j in range(have, need):
                entries[j] = free[len(free) - 1 - taken] if taken < len(free) else -1
                taken += 1
            tables[r][have:need] = entries[have:need]
        out.append((entries + [0] * width)[:width])
        cu.append(cu[-1] + n)
        for i in range(n):
            p = c + i
            pos.append(p)
            blk.append(entries[p // page] if p // page < need else -1)
            slot.append(p % page)
    pos, blk, slot = (x[:num_tokens] for x in (pos, blk, slot))
    pad = num_tokens - len(pos)
    left = None if free is None else len(free) - taken
    return (tables, out, cu, [max(0, c) + max(0, n) for c, n in zip(ctx, new)], pos + [0] * pad, blk + [-1] * pad,
            slot + [-1] * pad, left)


def _check(ctx, new, page, rows=None, table_rows=None, w=None, num_tokens=None, width=None, free=None, extra_free=0,
           seed=0):
    g = torch.Generator().manual_seed(seed)
    b = len(ctx)
    rows_ = list(range(b)) if rows is None else rows
    need = max([-(-(max(0, c) + max(0, n)) // page) for c, n in zip(ctx, new)], default=0)
    w = need + 2 if w is None else w
    tables = torch.randint(0, 1000, (table_rows or b, w), generator=g, dtype=torch.int32)
    width = w if width is None else width
    num_tokens = sum(max(0, n) for n in new) if num_tokens is None else num_tokens
    want = _host(tables.tolist(), rows_, ctx, new, page, num_tokens, width, free)
    dev = tables.to(DEV)
    kw = {}
    if free is not None:
        kw = {"free_blocks": _ints(free + [-5] * extra_free), "num_free": _ints([len(free)])}
    t = step_tables(dev, _ints(ctx), _ints(new), page, num_tokens, width=width,
                    rows=None if rows is None else _ints(rows), **kw)
    got = (dev.tolist(), t.block_tables.tolist(), t.cu_seqlens.tolist(), t.seq_lens.tolist(), t.positions.tolist(),
           t.block_mapping.tolist(), t.slot_mapping.tolist(), None if t.free_left is None else t.free_left.item())
    for name, x, y in zip(("tables", "block_tables", "cu_seqlens", "seq_lens", "positions", "block_mapping",
                           "slot_mapping", "free_left"), got, want):
        assert x == y, name
    assert all(x is None or x.dtype == torch.int32 for x in t)


@pytest.mark.parametrize("page", [1, 16, 24, 256])
@pytest.mark.parametrize("ctx,new", [
    ([0], [1]), ([5], [0]), ([15, 16, 17, 0], [1, 1, 1, 40]), ([0, 0, 0], [0, 0, 0]), ([300, 0, 1, 255], [0, 300, 0, 1]),
    ([-3, 10], [4, -2]), ([100] * 9, [1, 2, 3, 4, 5, 6, 7, 8, 9]),
])
def test_small(ctx, new, page):
    _check(ctx, new, page)
    _check(ctx, new, page, free=list(range(2000, 2900)), extra_free=7)
    _check(ctx, new, page, free=list(range(2000, 2900)), num_tokens=sum(max(0, n) for n in new) + 13, width=3)
    _check(ctx, new, page, rows=list(range(len(ctx) + 1, 1, -1)), table_rows=len(ctx) + 3, free=list(range(900)))


def test_a_list_that_is_too_short():
    for n in (0, 1, 3, 4, 5):
        _check([10, 16, 0, 31], [30, 1, 20, 2], 16, free=list(range(50, 50 + n)))


def test_tables_that_are_too_narrow_and_rows_that_are_not_there():
    _check([40, 3], [50, 60], 16, w=3, free=[1, 2, 3, 4, 5, 6, 7, 8])
    _check([40, 3], [50, 60], 16, w=3)
    _check([40, 3, 9], [50, 60, 20], 16, rows=[1, 7, -1], table_rows=2, free=[9, 8, 7, 6, 5, 4, 3])
    _check([40, 3], [5, 6], 16, w=0)
    _check([40, 3], [5, 6], 16, width=0)
    _check([40, 3, 70], [5, 6, 2], 16, num_tokens=7)  # fewer places than tokens
    _check([], [], 16, table_rows=3, w=4)


@pytest.mark.parametrize("b,lo,hi", [(1023, 0, 3), (1024, 1, 2), (2500, 0, 5), (5000, 0, 2)])
def test_many_requests(b, lo, hi):
    g = torch.Generator().manual_seed(b)
    ctx = torch.randint(0, 100, (b,), generator=g).tolist()
    new = torch.randint(lo, hi, (b,), generator=g).tolist()
    rows = torch.randperm(b + 10, generator=g)[:b].tolist()
    _check(ctx, new, 16, rows=rows, table_rows=b + 10, free=list(range(3 * b)), num_tokens=sum(new) + 5)


def test_many_tokens():
    _check([7, 100000, 3], [20000, 1, 30001], 16, free=list(range(9000)))
    _check([0], [70000], 256)


def test_large_lengths():
    """Sums past 31 bits saturate; tokens past the outputs and columns past the table are left out."""
    big = (1 << 30) - 1
    t = step_tables(torch.zeros(3, 4, dtype=torch.int32, device=DEV), _ints([big, big, 5]), _ints([big, big, big]), 16, 100)
    assert t.cu_seqlens.tolist() == [0, big, 2 * big, (1 << 31) - 1] and t.seq_lens.tolist() == [2 * big, 2 * big, big + 5]
    assert t.positions.tolist() == list(range(big, big + 100)) and set(t.block_mapping.tolist()) == {-1}


def test_strides_and_types():
    ctx, new = torch.tensor([[20, 0], [3, 0]], device=DEV), torch.tensor([[5, 9], [14, 9]], device=DEV)
    tables = torch.arange(64, dtype=torch.int32, device=DEV).view(8, 8).t()  # columns first
    t = step_tables(tables, ctx[:, 0], new[:, 0], 8, 19)
    assert t.block_tables.tolist() == [[0, 8, 16, 24, 0, 0, 0, 0], [1, 9, 17, 0, 0, 0, 0, 0]]
    assert t.block_mapping.tolist() == [16] * 4 + [24] + [1] * 5 + [9] * 8 + [17]


def test_graph_replays():
    """Steps of growing requests, the free list handed on: each replay as the eager call on the same inputs."""
    b, page = 6, 16
    ctx, new = torch.zeros(b, dtype=torch.int32, device=DEV), torch.zeros(b, dtype=torch.int32, device=DEV)
    tables = torch.zeros(b, 40, dtype=torch.int32, device=DEV)
    free, left = torch.arange(300, dtype=torch.int32, device=DEV), _ints([300])
    step_tables(tables, ctx, new, page, 128, free_blocks=free, num_free=left)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        t = step_tables(tables, ctx, new, page, 128, free_blocks=free, num_free=left)
        left.copy_(t.free_left)
    mine, mine_left = torch.zeros_like(tables), _ints([300])
    g = torch.Generator().manual_seed(1)
    for _ in range(5):
        lens = torch.randint(0, 20, (b,), generator=g).to(torch.int32).to(DEV)
        new.copy_(lens)
        graph.replay()
        want = step_tables(mine, ctx, lens, page, 128, free_blocks=free, num_free=mine_left)
        torch.cuda.synchronize()
        assert torch.equal(tables, mine) and all(torch.equal(x, y) for x, y in zip(t, want))
        mine_left = want.free_left
        ctx += lens
    used = tables[tables > 0].tolist()
    assert len(used) == len(set(used)) and 300 - mine_left.item() >= len(used)
