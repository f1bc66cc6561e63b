"""A step's tables for lengths past the range that they are taken within, [0, 2^30)."""

import pytest
import torch

from tinyserver_amd.kernels import step_tables

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("length", [(1 << 30) - 1, 1 << 30, (1 << 31) - 1, -1, -(1 << 31)])
@pytest.mark.parametrize("cached", [True, False])
def test_lengths_past_the_range(length, cached):
    longest = (1 << 30) - 1
    ctx, new = ([length, 3], [2, 4]) if cached else ([5, 3], [length, 4])
    ctx, new = (torch.tensor(x, dtype=torch.int32, device=DEV) for x in (ctx, new))
    t = step_tables(torch.zeros(2, 4, dtype=torch.int32, device=DEV), ctx, new, 16, 6)
    c, n = (x.clamp(0, longest).tolist() for x in (ctx, new))
    assert t.seq_lens.tolist() == [a + b for a, b in zip(c, n)] and t.cu_seqlens.tolist() == [0, n[0], n[0] + n[1]]
    want = [(c[0] + i) for i in range(min(n[0], 6))]
    want += [c[1] + i for i in range(6 - len(want))][: n[1]]
    assert t.positions.tolist() == want + [0] * (6 - len(want))
